// Attention of many new tokens over the paged cache (gfx950): chunks and prompts.
#include "cache_attention_device.hpp"

namespace q8 {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <bool H> __device__ __forceinline__ void mfma32(u32x4 a, u32x4 b, f32x16& c) {
    if constexpr (H) c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// A work-group of W waves has a tile of 32 W rows, 32 a wave, and takes 64 keys a step: keys and values go from
// memory to registers, and as 16-bit values to LDS while the step before them is computed, which has them once for all rows.
// Half of the waves do so for the values, the others for the keys.
// Keys lie in LDS by rows of a key's values, values by rows of one value's keys, both in pieces of 16 bytes whose place
// in the row is turned by the row's number, so that reads of 16 bytes down a column meet all banks.  The eight keys of a piece
// of the values are those that a lane has of each 16 after the scores (0-3, 8-11 and 4-7, 12-15).
// The scales come by the matrix cores too: a lane has one key's, as three BF16 terms, and their product with ones
// gives each lane those of the keys that it has after the scores.
template <int DT, int DP> struct Many {
    static constexpr int TERMS = DT == Q8_F32 ? 3 : 1, W = (int)many_rows(DT == Q8_F32, DP) / 32, THREADS = 64 * W;
    static constexpr bool QH = DT == Q8_F16, VH = DT != Q8_F32;
    static constexpr int KEY_UNITS = 64 * (DP / 16), KEY_LOADS = (KEY_UNITS + THREADS / 2 - 1) / (THREADS / 2);   // 16 bytes each
    static constexpr int VALUE_UNITS = 8 * (DP / 4), VALUE_LOADS = (VALUE_UNITS + THREADS / 2 - 1) / (THREADS / 2);  // eight keys of four values
    static constexpr int HELD = KEY_LOADS * 4 > VALUE_LOADS * 8 ? KEY_LOADS * 4 : VALUE_LOADS * 8;
    // bytes of LDS: keys and values twice
    static constexpr int KEY_ROW = DP * 2, VALUE_ROW = 128, KEYS = 64 * KEY_ROW, VALUES = DP * VALUE_ROW;
    // What a row turns its pieces by.  Reads of 16 bytes go by 16 lanes a cycle (0-3, 12-15, 20-27 and so on), writes by
    // eight, over 64 banks: rows of 256 bytes and more need 16 turns, of 128 eight for each of two rows, which bit 4
    // gives the writes of every fourth row too.
    static __device__ __forceinline__ uint32_t turn128(uint32_t row) { return ((row >> 1) & 7) ^ ((row >> 4) & 1); }
    static __device__ __forceinline__ uint32_t key_turn(uint32_t row) { return DP == 64 ? turn128(row) : row & 15; }
};

template <int DT, int DP> __global__ void __launch_bounds__((Many<DT, DP>::THREADS), (Many<DT, DP>::W / 4)) many_kernel(const AttentionArgs g) {
    typedef Many<DT, DP> F;
    typedef typename Type<DT>::T T;
    constexpr int TERMS = F::TERMS, S = DP / 16, D = DP / 32;
    __shared__ __attribute__((aligned(16))) char lds[2 * (F::KEYS + F::VALUES)];
    __shared__ uint64_t offsets[F::W][64];
    const Attention& a = g.a;
    const Paged& c = a.at;
    const uint32_t kv = blockIdx.x % c.heads, piece = blockIdx.y;
    Place t;
    // the last tiles of a sequence see the most keys and come first
    if (!find_tile(g, g.slots - 1 - blockIdx.x / c.heads, 32 * F::W, t)) return;
    const int pieces = max(1, pieces_of(t, g.piece));
    if ((int)piece >= pieces) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, half = lane >> 5;
    const int begin = t.begin + (int)(piece * g.piece), end = min(t.end, begin + (int)g.piece);

    // this lane's row; those past the tile's are its last
    const bool mine = wave * 32 + n < t.rows;
    const Row at = row_of(g, t, kv, min(wave * 32 + n, t.rows - 1));
    const int position = t.at + ((int)at.row - t.first);
    auto window_of = [&](int p) { return a.window && p - (int64_t)a.window + 1 > INT32_MIN ? (int)(p - (int64_t)a.window + 1) : INT32_MIN; };
    const int oldest = window_of(position);
    // of this wave's rows: the first's and the last's position (-1: no rows, nothing to compute)
    const int low = __builtin_amdgcn_readlane(position, 0), high = wave * 32 < t.rows ? __builtin_amdgcn_readlane(position, 31) : -1;
    const int all_from = window_of(high), none_to = window_of(low);

    u32x4 q[S][TERMS];
    {
        const T* row = (const T*)a.q + at.row * a.ldq + at.head * c.dim;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float v[8];
            query<DT>(row, s * 16 + half * 8, c.dim, v);
            terms_of<TERMS, F::QH>(v, q[s]);
        }
    }
    const float factor = a.scale * kLog2e;
    float R = kUnset, l = 0.0f;
    f32x16 o[D];
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;

    const int64_t head_rows = (int64_t)kv * c.page_tokens, page_rows = (int64_t)c.heads * c.page_tokens;
    // What the table says of this lane's key of the step from key k.  Not looked at before the step's loads: a wait for it
    // would be one for all loads before it.
    const int32_t* pages = c.table + (uint64_t)t.b * c.table_ld;
    auto page_of = [&](int k) __attribute__((always_inline)) { return pages[divide((uint32_t)min(k + lane, end - 1), c.page)]; };
    uint64_t* offset = offsets[wave];
    const bool values = wave < F::W / 2;
    const int worker = values ? tid : tid - F::THREADS / 2;
    uint32_t held[F::HELD];
    float k_scale = 0.0f, v_scale = 0.0f;
    // A step's loads; every wave finds all 64 keys for itself.  Rows of keys that are not there become those of one that
    // is; 0: none is.
    auto load = [&](int k, int page) __attribute__((always_inline)) {
        page = k + lane < end && (uint32_t)kept(page) < c.pages ? page : -1;
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
        if (values) {
#pragma unroll
            for (int x = 0; x < F::VALUE_LOADS; ++x) {
                const int u = worker + x * (F::THREADS / 2), part = u / (DP / 4) % 8, d = u % (DP / 4) * 4;
                const int first = part / 2 * 16 + part % 2 * 4;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    held[8 * x + e] = *reinterpret_cast<const uint32_t*>(c.v + offset[first + (e >> 2) * 8 + (e & 3)] + (d < (int)c.pitch ? d : 0));
            }
        } else {
#pragma unroll
            for (int x = 0; x < F::KEY_LOADS; ++x) {
                const int u = worker + x * (F::THREADS / 2), key_of = u / (DP / 16) % 64, d = u % (DP / 16) * 16;
                const u32x4 w = *reinterpret_cast<const u32x4*>(c.k + offset[key_of] + (d < (int)c.pitch ? d : 0));
#pragma unroll
                for (int e = 0; e < 4; ++e) held[4 * x + e] = w[e];
            }
        }
        __builtin_amdgcn_wave_barrier();
        return there;
    };
    auto store = [&](int to) __attribute__((always_inline)) {
        if (values) {
#pragma unroll
            for (int x = 0; x < F::VALUE_LOADS; ++x) {
                const int u = worker + x * (F::THREADS / 2), part = u / (DP / 4), d = u % (DP / 4) * 4;
                if (F::VALUE_UNITS % (F::THREADS / 2) && u >= F::VALUE_UNITS) break;
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = kept(held[8 * x + e]);
                u32x4 r[4];
                columns<F::VH>(w, r);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *reinterpret_cast<u32x4*>(lds + 2 * F::KEYS + to * F::VALUES + (d + j) * F::VALUE_ROW + (part ^ F::turn128(d + j)) * 16) = r[j];
            }
        } else {
#pragma unroll
            for (int x = 0; x < F::KEY_LOADS; ++x) {
                const int u = worker + x * (F::THREADS / 2), key_of = u / (DP / 16), part = u % (DP / 16) * 2;
                if (F::KEY_UNITS % (F::THREADS / 2) && u >= F::KEY_UNITS) break;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x2 w0 = four<F::QH>(kept(held[4 * x + 2 * h])), w1 = four<F::QH>(kept(held[4 * x + 2 * h + 1]));
                    *reinterpret_cast<u32x4*>(lds + to * F::KEYS + key_of * F::KEY_ROW + ((part + h) ^ F::key_turn(key_of)) * 16) =
                        u32x4{w0[0], w0[1], w1[0], w1[1]};
                }
            }
        }
    };
    // three terms of this lane's key's scale, and those for the half of the lanes that has the keys of half step i, zeros for the other
    auto split = [&](float x) __attribute__((always_inline)) {
        uint32_t b[3];
        three(x, b);
        return u32x2{uppers(b[0], b[1]), b[2] >> 16};
    };
    auto terms_in = [&](u32x2 x, int i) __attribute__((always_inline)) {
        const bool on = half == i;
        return u32x4{on ? x[0] : 0u, on ? x[1] : 0u, 0u, 0u};
    };
    const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0, 0};
    // where this lane reads: a place's piece is turned by what the row's number turns, so another piece is an exclusive or away
    const uint32_t key_at = n * F::KEY_ROW + ((half ^ F::key_turn(n)) * 16);
    const uint32_t value_at = 2 * F::KEYS + n * F::VALUE_ROW + ((half ^ F::turn128(n)) * 16);
    // 32 keys from k, the i-th half of a step's
    auto compute = [&](int from, int i, int k, uint32_t there, u32x2 sk_mine, u32x2 sv_mine) __attribute__((always_inline)) {
        if (!there || k > high || k + 31 < none_to) return;
        f32x16 score, sk, sv;
#pragma unroll
        for (int e = 0; e < 16; ++e) score[e] = sk[e] = sv[e] = 0.0f;
        constexpr int AT_ONCE = S < 8 ? S : 8;
#pragma unroll
        for (int s0 = 0; s0 < S; s0 += AT_ONCE) {
            u32x4 w[AT_ONCE];
#pragma unroll
            for (int s = 0; s < AT_ONCE; ++s)
                w[s] = *reinterpret_cast<const u32x4*>(lds + from * F::KEYS + i * 32 * F::KEY_ROW + (key_at ^ ((s0 + s) * 32)));
            __builtin_amdgcn_sched_barrier(0);
            if (s0 == 0) {
                mfma32<false>(terms_in(sk_mine, i), ones, sk);
                mfma32<false>(terms_in(sv_mine, i), ones, sv);
            }
#pragma unroll
            for (int s = 0; s < AT_ONCE; ++s)
#pragma unroll
                for (int m = 0; m < TERMS; ++m) mfma32<F::QH>(w[s], q[s0 + s][m], score);
        }
        const bool whole = there == 0xffffffffu && k + 31 <= low && k >= all_from;
        uint32_t seen = 0xffff;
        if (!whole) {
            seen = 0;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int x = (e >> 2) * 8 + half * 4 + (e & 3);
                const bool on = (there >> x & 1) && k + x <= position && k + x >= oldest;
                seen |= on ? 1u << e : 0u;
                if (!on) {      // weights of 0, whatever the scales
                    score[e] = -__builtin_huge_valf();
                    sk[e] = 1.0f;
                    sv[e] = 0.0f;
                }
            }
        }
        float p[16], w[16], top = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[e], sk[e], -R));
            w[e] = p[e] * sv[e];
            top = e ? fmaxf(top, fabsf(w[e])) : fabsf(w[e]);
        }
        if (__any(!(top <= kTop))) {
            float most = kUnset;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (seen >> e & 1)
                    most = fmaxf(most, __builtin_fmaf(score[e], sk[e], __builtin_amdgcn_logf(fmaxf(fabsf(sv[e]), 0x1p-100f))));
            most = fmaxf(most, __shfl_xor(most, 32));
            const float next = most > R + kRoom ? most - kRoom : R;
            const float down = __builtin_amdgcn_exp2f(R - next);
            R = next;
            l *= down;
#pragma unroll
            for (int d = 0; d < D; ++d) o[d] *= down;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[e], sk[e], -R));
                w[e] = p[e] * sv[e];
            }
        }
        u32x4 weight[2][TERMS];
#pragma unroll
        for (int e = 0; e < 16; ++e) l += p[e];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float x[8] = {w[8 * j], w[8 * j + 1], w[8 * j + 2], w[8 * j + 3], w[8 * j + 4], w[8 * j + 5], w[8 * j + 6], w[8 * j + 7]};
            terms_of<TERMS, F::VH>(x, weight[j]);
        }
        constexpr int D_AT_ONCE = D < 4 ? D : 4;
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += D_AT_ONCE) {
            u32x4 v[D_AT_ONCE][2];
#pragma unroll
            for (int d = 0; d < D_AT_ONCE; ++d)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    v[d][j] = *reinterpret_cast<const u32x4*>(lds + from * F::VALUES + (value_at ^ (i * 64 + j * 32)) + (d0 + d) * 32 * F::VALUE_ROW);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int d = 0; d < D_AT_ONCE; ++d)
#pragma unroll
                    for (int m = 0; m < TERMS; ++m) mfma32<F::VH>(v[d][j], weight[j][m], o[d0 + d]);
        }
    };

    // Steps in flight: the one that is computed, the next one in LDS or on its way there, the one after in registers.
    // Half of the waves store and load before they compute, the others after, so that of the two on a SIMD one has
    // conversions for the vector unit while the other has products.
    constexpr int STEP = 64;
    uint64_t there = 0, there1 = 0, there2 = 0;
    float sk = 0.0f, sv = 0.0f, sk1 = 0.0f, sv1 = 0.0f;
    int page = 0;
    if (begin < end) {
        there = load(begin, page_of(begin));
        sk = k_scale;
        sv = v_scale;
        if (there) store(0);
        there1 = load(begin + STEP, page_of(begin + STEP));
        sk1 = k_scale;
        sv1 = v_scale;
        page = page_of(begin + 2 * STEP);
    }
    int buffer = 0;
    for (int k = begin; k < end; k += STEP, buffer ^= 1) {
        __syncthreads();        // this step is in LDS, and the one before is done with its half of it
        auto forward = [&]() __attribute__((always_inline)) {
            if (there1) store(buffer ^ 1);
            there2 = load(k + 2 * STEP, page);
            page = page_of(k + 3 * STEP);
        };
        if (!values) forward();
        const u32x2 ks = split(sk * factor), vs = split(sv);
        compute(buffer, 0, k, (uint32_t)there, ks, vs);
        compute(buffer, 1, k + 32, (uint32_t)(there >> 32), ks, vs);
        if (values) forward();
        there = there1;
        there1 = there2;
        sk = sk1;
        sv = sv1;
        sk1 = k_scale;
        sv1 = v_scale;
    }

    l += __shfl_xor(l, 32);
    if (!mine) return;
    const uint64_t to = at.row * a.heads + at.head;
    if (pieces > 1) {       // join_kernel's
        const uint64_t own = (uint64_t)piece * c.tokens * a.heads + to;
#pragma unroll
        for (int d = 0; d < D; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<f32x4*>(g.sums + own * DP + d * 32 + i * 2 + half * 4) = f32x4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
        if (half == 0) {
            g.stats[2 * own] = R;
            g.stats[2 * own + 1] = l;
        }
        return;
    }
    const float part = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = (T*)a.out + at.row * a.ldo + at.head * c.dim;
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t x = d * 32 + (i >> 2) * 8 + half * 4 + (i & 3);
            if (x < c.dim) Type<DT>::put(out + x, o[d][i] * part);
        }
    if (a.lse && half == 0) a.lse[to] = l == 0.0f ? -__builtin_huge_valf() : (R + __builtin_log2f(l)) * kLn2;
}

// The pieces' sums of a tile's rows: DP / 8 threads a row, 2048 / DP rows a work-group.  (A work-group of the kernel before
// that finishes a tile and adds them alone reads for longer than all work-groups together: 64 tokens over 8192 keys,
// 32 pieces, 195 us.)
template <int DT, int DP> __global__ void __launch_bounds__(256) join_kernel(const AttentionArgs g) {
    typedef typename Type<DT>::T T;
    constexpr int ACROSS = DP / 8;
    const Attention& a = g.a;
    const Paged& c = a.at;
    const uint32_t kv = blockIdx.x % c.heads;
    Place t;
    if (!find_tile(g, g.slots - 1 - blockIdx.x / c.heads, 32 * Many<DT, DP>::W, t)) return;
    const int pieces = pieces_of(t, g.piece), r = blockIdx.y * (256 / ACROSS) + threadIdx.x / ACROSS, d = threadIdx.x % ACROSS * 8;
    if (pieces <= 1 || r >= t.rows) return;
    const Row at = row_of(g, t, kv, r);
    const uint64_t stride = (uint64_t)c.tokens * a.heads, to = at.row * a.heads + at.head;
    float R = kUnset, l = 0.0f, v[8] = {};
    constexpr int AHEAD = 4;
    for (int p = 0; p < pieces; p += AHEAD) {
        float o[AHEAD][8], rp[AHEAD], lp[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const uint64_t from = to + (uint64_t)min(p + i, pieces - 1) * stride;
            rp[i] = g.stats[2 * from];
            lp[i] = g.stats[2 * from + 1];
            Type<Q8_F32>::load8(g.sums + from * DP + d, o[i]);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (p + i < pieces) add_part(R, l, v, rp[i], lp[i], o[i]);
    }
    const float part = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= part;
    if (d < (int)c.dim) store_part<DT>((T*)a.out + at.row * a.ldo + at.head * c.dim, d, c.dim, v);
    if (a.lse && d == 0) a.lse[to] = l == 0.0f ? -__builtin_huge_valf() : (R + __builtin_log2f(l)) * kLn2;
}

template <int DT, int DP> hipError_t run(const AttentionArgs& g, uint32_t pieces, hipStream_t s) {
    void* args[] = {const_cast<AttentionArgs*>(&g)};
    typedef Many<DT, DP> F;
    const uint32_t tiles = g.slots * g.a.at.heads;
    const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(&many_kernel<DT, DP>), dim3(tiles, pieces), dim3(F::THREADS), args, 0, s);
    if (e != hipSuccess || pieces == 1) return e;
    return hipLaunchKernel(reinterpret_cast<const void*>(&join_kernel<DT, DP>), dim3(tiles, 32 * F::W * DP / 2048), dim3(256), args, 0, s);
}

}  // namespace

hipError_t launch_many(int dtype, const AttentionArgs& g, uint32_t pieces, hipStream_t s) {
    return for_head(dtype, g.a.at.dim, [&](auto dt, auto dp) { return run<decltype(dt)::value, decltype(dp)::value>(g, pieces, s); });
}

hipError_t prepare_many() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(&many_kernel<Q8_F32, 64>));
}

}  // namespace q8
