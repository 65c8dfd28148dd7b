// Attention of many new tokens over the paged cache (gfx950): chunks and prompts.
#include "cache_image.hpp"

namespace q8 {
namespace {

template <bool H> __device__ __forceinline__ void mfma32(u32x4 a, u32x4 b, f32x16& c) {
    if constexpr (H) c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// A work-group of W waves has a tile of 32 W rows, 32 a wave, and takes 64 keys a step, whose image it makes itself in LDS: half
// of the waves load and convert the values, the others the keys, while steps before are computed.  Bounded by the latency of few
// work-groups' steps (64 tokens of 32 heads of 128 over 8192 keys, BF16: 41 us; 5 chunks of up to 77 over 1501, FP32: 20.9).  FP32
// takes three products for one and leaves a SIMD one wave (400 registers; 512 tokens over 2048 keys 84 us, the products alone
// 38; a prompt of 2048 169 and 86).  Heads of 256 spill registers, FP32 134 and 16-bit types 9 (BF16, 16 heads, 1024 tokens over
// 4096 keys: 173 us, the products 50).
template <int DT, int DP> struct Many : Image<DT, DP> {
    static constexpr int TERMS = DT == Q8_F32 ? 3 : 1, W = (int)many_rows(DT == Q8_F32, DP) / 32, THREADS = 64 * W;
};

template <int DT, int DP>
__global__ void __launch_bounds__((Many<DT, DP>::THREADS), (Many<DT, DP>::W / 4)) many_kernel(const AttentionArgs g) {
    typedef Many<DT, DP> F;
    typedef Units<DT, DP, F::THREADS / 2> U;
    typedef typename Type<DT>::T T;
    constexpr int TERMS = F::TERMS, S = DP / 16, D = DP / 32, STEP = 64;
    // A step's last values are multiplied after the next one's first keys, so its image stays for that long, while the
    // next one but one's comes.  Heads of 256 values leave room for two images, and wait.
    constexpr int IMAGES = DP == 256 ? 2 : 3;
    constexpr bool CARRY = IMAGES > 2;
    __shared__ __attribute__((aligned(1024))) char lds[IMAGES * F::BYTES];
    __shared__ uint64_t offsets[F::W][64];
    __shared__ Far fars[F::W][32];
    const Attention& a = g.a;
    const Paged& c = a.at;
    const uint32_t kv = blockIdx.x % c.heads, piece = blockIdx.y;
    Place t;
    if (!find_rows<32 * F::W>(g, t)) return;
    const int pieces = max(1, pieces_of(t, g.piece));
    if ((int)piece >= pieces) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, half = lane >> 5;
    const int begin = t.begin + (int)(piece * g.piece), end = piece_end(t, begin, g.piece);

    // this lane's row; those past the tile's are its last
    const bool mine = wave * 32 + n < t.rows;
    const int in_tile = min(wave * 32 + n, t.rows - 1);
    const int position = t.at + (int)divide((uint32_t)(t.row + in_tile), g.by_group);
    auto window_of = [&](int p) { return a.window && p - (int64_t)a.window + 1 > INT32_MIN ? (int)(p - (int64_t)a.window + 1) : INT32_MIN; };
    const int oldest = window_of(position);
    // of this wave's rows: the first's and the last's position (-1: no rows, nothing to compute)
    const int low = __builtin_amdgcn_readlane(position, 0), high = wave * 32 < t.rows ? __builtin_amdgcn_readlane(position, 31) : -1;
    const int all_from = window_of(high), none_to = window_of(low);

    u32x4 q[S][TERMS];
    {
        const Row at = row_of(g, t, kv, in_tile);
        const T* row = (const T*)a.q + at.row * a.ldq + at.head * c.dim;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float v[8];
            query<DT>(row, s * 16 + half * 8, c.dim, v);
            terms_of<TERMS, F::QH>(v, q[s]);
        }
    }
    float R = kUnset, l = 0.0f;
    f32x16 o[D];
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;

    const uint32_t key_at = F::key_at(n, half), value_at = F::value_at(n, half);
    // Fragments of a half step's keys and values, as many at a time as there are registers for.
    constexpr int KF = S < 8 ? S : 8, VF = D / 2;
    u32x4 kf[KF], vf[VF][2];
    auto read_keys = [&](int from, int i, int s0) __attribute__((always_inline)) {
        const uint32_t base = kept(key_at + from * F::BYTES);
#pragma unroll
        for (int s = 0; s < KF; ++s) kf[s] = *reinterpret_cast<const u32x4*>(lds + base + (s0 + s) * 32 + i * 32 * F::KEY_ROW);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto read_values = [&](int from, int i, int part) __attribute__((always_inline)) {
        const uint32_t base = kept(value_at + from * F::BYTES);
#pragma unroll
        for (int d = 0; d < VF; ++d)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                vf[d][j] = *reinterpret_cast<const u32x4*>(lds + base + i * 64 + j * 32 + (part * VF + d) * 32 * F::VALUE_ROW);
        __builtin_amdgcn_sched_barrier(0);
    };
    // whether a half step's 32 keys from k are seen by a row of this wave
    auto needed = [&](int k, uint32_t there) __attribute__((always_inline)) { return there && k <= high && k + 31 >= none_to; };
    f32x16 score;
    u32x4 weight[2][TERMS];
    auto multiply = [&](int part) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int d = 0; d < VF; ++d)
#pragma unroll
                for (int m = 0; m < TERMS; ++m) mfma32<F::VH>(vf[d][j], weight[j][m], o[part * VF + d]);
    };
    // The products of a half step: the weights of the one before (`old`, half `pi` of LDS `pfrom`) with its values, and the scores of
    // this one (`now`, half i of LDS `from`).
    auto products = [&](bool old, int pfrom, int pi, bool now, int from, int i) __attribute__((always_inline)) {
        if (old) read_values(pfrom, pi, 0);
        if (now) read_keys(from, i, 0);
        if (old) {
            multiply(0);
            read_values(pfrom, pi, 1);
        }
        if (now) {
#pragma unroll
            for (int e = 0; e < 16; ++e) score[e] = 0.0f;
#pragma unroll
            for (int s0 = 0; s0 < S; s0 += KF) {
                if (s0) read_keys(from, i, s0);
#pragma unroll
                for (int s = 0; s < KF; ++s)
#pragma unroll
                    for (int m = 0; m < TERMS; ++m) mfma32<F::QH>(kf[s], q[s0 + s][m], score);
            }
        }
        if (old) multiply(1);
    };
    // The weights of 32 keys from k.  The scales are read again where R moves, which is seldom: kept until then they
    // and what they were multiplied with are more registers than there are.
    auto weights = [&](int from, int i, int k, uint32_t there) __attribute__((always_inline)) {
        const uint32_t scale_at = (uint32_t)(from * F::BYTES + F::SCALES + (i * 32 + 4 * half) * 4);
        auto scales_of = [&](uint32_t at, int e, f32x4& x, f32x4& y) __attribute__((always_inline)) {
            x = *reinterpret_cast<const f32x4*>(lds + at + 8 * e);
            y = *reinterpret_cast<const f32x4*>(lds + at + 256 + 8 * e);
        };
        const bool whole = there == 0xffffffffu && k + 31 <= low && k >= all_from;
        uint32_t seen = 0xffff;
        if (!whole) {
            // bits 8 q + 4 half + z, of keys up to this row's position and from its window's first
            const int to = position < k ? 0 : min(position - k + 1, 32), from = oldest > k ? min(oldest - k, 32) : 0;
            uint32_t mask = there & (uint32_t)((1ull << to) - 1) & ~(uint32_t)((1ull << from) - 1);
            mask >>= 4 * half;
            seen = (mask & 0xf) | (mask >> 4 & 0xf0) | (mask >> 8 & 0xf00) | (mask >> 12 & 0xf000);
        }
        float w[16], sum = 0.0f, top = 0.0f;
        auto weigh = [&](auto all, auto exponent_of) __attribute__((always_inline)) {
            const uint32_t at = kept(scale_at);
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                f32x4 sk, sv;
                scales_of(at, e, sk, sv);
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const bool on = all.value || (seen >> (e + z) & 1);
                    float p = __builtin_amdgcn_exp2f(exponent_of(score[e + z], sk[z]));
                    p = on ? p : 0.0f;
                    w[e + z] = on ? p * sv[z] : 0.0f;
                    sum = e + z ? sum + p : p;
                    top = e + z ? fmaxf(top, fabsf(w[e + z])) : fabsf(w[e + z]);
                }
            }
        };
        auto less_R = [&](float t, float k) __attribute__((always_inline)) { return __builtin_fmaf(t, k, -R); };
        if (whole) weigh(Int<1>{}, less_R);
        else weigh(Int<0>{}, less_R);
        // (a product with a scale of 0 may be no number, which fmaxf passes over; the exponential then is infinite)
        if (__any(!(top <= kTop) || !(l + sum <= kMostSum))) {
            Reference r(R, &fars[wave][kept((uint32_t)n)]);
            const float down = moved<32>(r, l, kRoom, [&](auto each) __attribute__((always_inline)) {
                const uint32_t at = kept(scale_at), mask = kept(seen);
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    f32x4 sk, sv;
                    scales_of(at, e, sk, sv);
#pragma unroll
                    for (int z = 0; z < 4; ++z) each(mask >> (e + z) & 1, score[e + z], sk[z], sv[z]);
                    if (e == 4) __builtin_amdgcn_sched_barrier(0);      // half of the scales in registers at a time
                }
            });
            R = r.R;
            r.keep(&fars[wave][kept((uint32_t)n)]);
            l *= down;
#pragma unroll
            for (int d = 0; d < D; ++d) o[d] *= down;
            if (__builtin_expect(__any(r.is_far()), 0)) {
                const Reference wide(R, &fars[wave][kept((uint32_t)n)]);
                weigh(Int<0>{}, [&](float t, float k) __attribute__((always_inline)) { return exponent(wide, t, k); });
            } else {
                weigh(Int<0>{}, less_R);
            }
        }
        l += sum;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float x[8] = {w[8 * j], w[8 * j + 1], w[8 * j + 2], w[8 * j + 3], w[8 * j + 4], w[8 * j + 5], w[8 * j + 6], w[8 * j + 7]};
            terms_of<TERMS, F::VH>(x, weight[j]);
        }
    };

    // A step: `here` its keys that are there, in LDS `from`; `old`: weights wait for the last values of the step before, in LDS `before`.
    bool old = false;
    auto step = [&](int k, uint64_t here, int from, int before) __attribute__((always_inline)) {
        const uint32_t lower = (uint32_t)here, upper = (uint32_t)(here >> 32);
        const bool first = needed(k, lower), second = needed(k + 32, upper);
        products(old, before, 1, first, from, 0);
        if (first) weights(from, 0, k, lower);
        products(first, from, 0, second, from, 1);
        if (second) weights(from, 1, k + 32, upper);
        old = second;
        if (!CARRY) {
            products(old, from, 1, false, 0, 0);
            old = false;
        }
    };
    int last = 0;       // the last step's image
    // What the table says of this lane's key of the step from key k.  Not looked at before the step's loads: a wait for it
    // would be one for all loads before it.
    const int32_t* pages = c.table + (uint64_t)t.b * c.table_ld;
    auto page_of = [&](int k) __attribute__((always_inline)) { return pages[divide((uint32_t)min(k + lane, end - 1), c.page)]; };
    const bool values = wave < F::W / 2;
    const int worker = values ? tid : tid - F::THREADS / 2;
    const uint32_t at = values ? U::value_at(worker) : U::key_at(worker);
    uint32_t held[U::HELD];
    float scale = 0.0f;     // wave 0 has the values', wave W / 2 the keys'
    // A step's loads; every wave finds all 64 keys for itself.
    auto load = [&](int k, int page) __attribute__((always_inline)) {
        int64_t row;
        const uint64_t there = find_row(c, kv, k, end, page, row);
        if (!there) return there;
        if (wave == 0) scale = c.v_scale[row];
        if (wave == F::W / 2) scale = c.k_scale[row];
        offsets[wave][lane] = (uint64_t)row * c.pitch;
        __builtin_amdgcn_wave_barrier();
        if (values) U::load_values(c, offsets[wave], worker, held);
        else U::load_keys(c, offsets[wave], worker, held);
        __builtin_amdgcn_wave_barrier();
        return there;
    };
    auto store = [&](int to) __attribute__((always_inline)) {
        char* image = lds + to * F::BYTES;
        const uint32_t place = kept(at);
        if (wave == 0) *reinterpret_cast<float*>(image + F::SCALES + 256 + lane * 4) = scale;
        if (wave == F::W / 2) *reinterpret_cast<float*>(image + F::SCALES + lane * 4) = scale * (a.scale * kLog2e);
        if (values) U::store_values(image, place, worker, held);
        else U::store_keys(image, place, worker, held);
    };
    // Steps in flight: the one that is computed, the next one in LDS or on its way there, the one after in registers.
    // Half of the waves store and load before they compute, the others after, so that of the two on a SIMD one has
    // conversions for the vector unit while the other has products.
    uint64_t there = 0, there1 = 0, there2 = 0;
    int page = 0;
    if (begin < end) {
        there = load(begin, page_of(begin));
        if (there) store(0);
        there1 = load(begin + STEP, page_of(begin + STEP));
        page = page_of(begin + 2 * STEP);
    }
    int from = 0;
    for (int k = begin; k < end; k += STEP) {
        const int next = from + 1 == IMAGES ? 0 : from + 1, before = from ? from - 1 : IMAGES - 1;
        __syncthreads();        // this step is in LDS, and all are done with the image that the next one goes to
        auto forward = [&]() __attribute__((always_inline)) {
            if (there1) store(next);
            there2 = load(k + 2 * STEP, page);
            page = page_of(k + 3 * STEP);
        };
        if (!values) forward();
        step(k, there, from, before);
        if (values) forward();
        there = there1;
        there1 = there2;
        last = from;
        from = next;
    }
    if (CARRY) products(old, last, 1, false, 0, 0);

    l += __shfl_xor(l, 32);
    if (!mine) return;
    put_row<DT, DP>(g, row_of(g, t, kv, (int)kept((uint32_t)in_tile)), piece, pieces, half, Reference(R, &fars[wave][n]), l, o);
}

template <int DT, int DP> hipError_t run(const AttentionArgs& g, uint32_t pieces, hipStream_t s) {
    typedef Many<DT, DP> F;
    const uint32_t tiles = g.slots * g.a.at.heads;
    const hipError_t e = launch(&many_kernel<DT, DP>, dim3(tiles, pieces), F::THREADS, g, s);
    if (e != hipSuccess || pieces == 1) return e;
    return launch(&join_kernel<DT, DP, 32 * F::W>, dim3(tiles, 32 * F::W * DP / 2048), 256, g, s);
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
