// Gradients from operands as they are (gfx950): D (rows x cols) = sum over s of A_s,row scale_s q_s,col.
//
// A matrix instruction's operand is eight consecutive values of the summed index a lane, and q (and
// dy, for the gradient of the weights) has that index from row to row.  A lane that takes
// eight rows of W values each has W such operands after a turn in registers, so a wave
// turns what it multiplies, and nothing is laid out in memory first: one launch and no
// workspace.  That turn is done again by each work-group that reads the values, so it pays for
// small gradients, where launches and their latency count: BF16 512^3 6.0 us (8.0 with the 16-bit operand
// turned), laid out and multiplied 12.0 (12.5); 1024^3 9.0 (11.1) and 15.8 (17.6).  About 3 us (4 turned) are the
// launch, the first loads and the join; then each step waits for its loads, 0.75 us (1.0) with one
// work-group a CU, and 1.3 - 1.75 for both of two, where the loads' number bounds it.  FP32 takes three times
// the matrix instructions and 400 to 700 others a step to split 32 (64) values a lane into three terms, which
// bound it: 512^3 8.9 us (13.1).  Groups in XCD order: 4096 x 1024 x 1024 25 -> 21 us.
#include "q8_device.hpp"
#include "q8_internal.hpp"
#include "q8_plan.hpp"

namespace q8 {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef u32x2 u32x2_at2 __attribute__((aligned(2)));

template <bool HALF> __device__ __forceinline__ void mfma(u32x4 a, u32x4 b, f32x4& c) {
    if constexpr (HALF)
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ u32x4 zero8(u32x4) { return u32x4{0, 0, 0, 0}; }
__device__ __forceinline__ Type<Q8_F32>::Eight zero8(const Type<Q8_F32>::Eight&) {
    return {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
}

// Eight values as they are loaded.
template <typename EIGHT, bool ODD> struct Piece { typedef EIGHT T; };
template <typename EIGHT> struct Piece<EIGHT, true> { typedef Raw<true>::T T; };

// Four results of a row; the first `skip` of them are another lane's.
template <int DT>
__device__ __forceinline__ void put4(typename Type<DT>::T* y, f32x4 v, uint32_t skip, bool accumulate) {
    if (accumulate) {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if (e >= skip) v[e] += Type<DT>::get(y + e);
    }
    if (skip) {
#pragma unroll
        for (uint32_t e = 1; e < 4; ++e)
            if (e >= skip) Type<DT>::put(y + e, v[e]);
    } else if constexpr (DT == Q8_F32) {
        *reinterpret_cast<f32x4_at4*>(y) = v;
    } else {
        *reinterpret_cast<u32x2_at2*>(y) = u32x2{Type<DT>::pair(v[0], v[1]), Type<DT>::pair(v[2], v[3])};
    }
}

// A work-group has 64 rows and 64 columns; its waves take steps of 32 values of the summed index in
// turn, a step's loads in flight while the one before is multiplied, and add their sums in LDS.
// TURN: A has the summed index from row to row too, a lane takes eight values of a row, and a
// work-group has 128 rows.
// ODD (not turned): rows of 16-bit values that start between dwords, see Raw.
template <int DT, bool TURN, int WAVES, bool ODD>
__global__ void __launch_bounds__(WAVES * 64, DT == Q8_F32 && TURN ? 1 : 2) gradient_kernel(const Gradient p) {
    constexpr int MT = kGradientRows[TURN] / 16, NT = 4, TERMS = DT == Q8_F32 ? 3 : 1;
    constexpr bool HALF = DT == Q8_F16;
    typedef typename Type<DT>::T T;
    typedef typename Type<DT>::Eight Eight;
    __shared__ f32x4 red[WAVES][4 * NT][64];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t fr = lane & 15, fg = lane >> 4;
    const uint32_t across = (p.cols + 16 * NT - 1) / (16 * NT);
    const uint32_t z = xcd_order(blockIdx.x, gridDim.x);
    const uint32_t row0 = z / across * (16 * MT), col0 = z % across * (16 * NT);

    float down = 1.0f, up = 1.0f;
    if constexpr (HALF) powers(largest<WAVES * 64>(p.scale, p.sum, *reinterpret_cast<uint32_t(*)[WAVES]>(&red[0][0][0])), down, up);

    // The last values of a row are taken with those before them, which are not stored twice.
    const uint32_t c = min(col0 + fr * 4, p.cols - 4);
    const uint32_t r = TURN ? min(row0 + fr * 8, p.rows - 8) : 0;
    const T* const a = (const T*)p.a + r;
    uint32_t rows[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) rows[i] = min(row0 + i * 16 + fr, p.rows - 1);
    struct Step {
        typename Piece<Eight, ODD>::T a[MT];
        uint32_t at[ODD ? MT : 1];
        uint32_t q[8];
        float s[8];
    };
    auto fetch = [&](Step& v, uint32_t s0) __attribute__((always_inline)) {
        uint32_t s = s0 + fg * 8;
        const bool whole = s0 + 32 <= p.sum;
        if (whole) {
            const f32x4 lo = *reinterpret_cast<const f32x4_at4*>(p.scale + s), hi = *reinterpret_cast<const f32x4_at4*>(p.scale + s + 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) { v.s[k] = lo[k]; v.s[4 + k] = hi[k]; }
        } else {
            // the last step: as far back as it is whole, and zeros for what has been
            if constexpr (!TURN) s = p.sum - 32 + fg * 8;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t at = s + k;
                v.s[k] = at >= s0 && at < p.sum ? p.scale[min(at, p.sum - 1)] : 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            v.q[k] = *reinterpret_cast<const u32_at1*>(p.q + (uint64_t)min(s + k, p.sum - 1) * p.ldq + c);
        if constexpr (TURN) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v.a[k] = Type<DT>::get8(a + (uint64_t)min(s + k, p.sum - 1) * p.lda);
            if (!whole) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (s + k >= p.sum) v.a[k] = zero8(v.a[k]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const T* from = a + rows[i] * p.lda + s;
                if constexpr (ODD) {
                    v.at[i] = whole ? (uint32_t)(uintptr_t)from & 3u : 0u;
                    if (whole) v.a[i] = Raw<true>::load((const char*)from);
                    else v.a[i].w = Type<DT>::get8(from);
                } else {
                    v.a[i] = Type<DT>::get8(from);
                }
            }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (s + e >= s0) continue;
                        if constexpr (ODD) v.a[i].w[e / 2] &= e % 2 ? 0x0000ffffu : 0xffff0000u;
                        else if constexpr (DT != Q8_F32) v.a[i][e / 2] &= e % 2 ? 0x0000ffffu : 0xffff0000u;
                        else if (e < 4) v.a[i].lo[e % 4] = 0.0f;
                        else v.a[i].hi[e % 4] = 0.0f;
                    }
            }
        }
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    auto multiply = [&](const Step& v) __attribute__((always_inline)) {
        u32x4 b[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float x[8];
            // a scale that is not a number takes its whole row along, zeros too
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                x[k] = (float)(int8_t)(v.q[k] >> (8 * j));
                if constexpr (DT != Q8_F32) x[k] *= HALF ? v.s[k] * down : v.s[k];
            }
            b[j] = u32x4{pair16<HALF>(x[0], x[1]), pair16<HALF>(x[2], x[3]), pair16<HALF>(x[4], x[5]), pair16<HALF>(x[6], x[7])};
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            u32x4 w[TERMS];
            if constexpr (DT == Q8_F32) {
                uint32_t h[8][3];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const Eight& from = v.a[TURN ? k : i];
                    const int e = TURN ? i : k;
                    three((e < 4 ? from.lo[e % 4] : from.hi[e % 4]) * v.s[k], h[k]);
                }
#pragma unroll
                for (int t = 0; t < TERMS; ++t)
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[t][k] = uppers(h[2 * k][t], h[2 * k + 1][t]);
            } else if constexpr (TURN) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    w[0][k] = __builtin_amdgcn_perm(v.a[2 * k + 1][i / 2], v.a[2 * k][i / 2], i % 2 ? 0x07060302u : 0x05040100u);
            } else if constexpr (ODD) {
                w[0] = Raw<true>::value(v.a[i], v.at[i]);
            } else {
                w[0] = v.a[i];
            }
#pragma unroll
            for (int t = 0; t < TERMS; ++t)
#pragma unroll
                for (int j = 0; j < NT; ++j) mfma<HALF>(w[t], b[j], acc[i][j]);
        }
    };
    Step v0, v1;
    uint32_t s0 = wave * 32;
    if (s0 < p.sum) fetch(v0, s0);
#pragma unroll 1
    while (s0 < p.sum) {
        s0 += WAVES * 32;
        if (s0 < p.sum) fetch(v1, s0);
        multiply(v0);
        v0 = v1;    // (two copies of the loop would hold two sets of sums)
    }
    const uint32_t skip = col0 + fr * 4 - c;    // 4 and more: no column is this lane's
#pragma unroll
    for (int h = 0; h < MT / 4; ++h) {
        __syncthreads();    // (and the scales' maxima have been read)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) red[wave][i * NT + j][lane] = acc[h * 4 + i][j];
        __syncthreads();
        f32x4 sum[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            sum[j] = red[0][wave % 4 * NT + j][lane];
#pragma unroll
            for (int k = 1; k < WAVES; ++k) sum[j] += red[k][wave % 4 * NT + j][lane];
        }
        const uint32_t i = h * 4 + wave % 4;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            if (WAVES == 8 && k / 2 != wave / 4) continue;      // four rows, of which two waves store two each
            const uint32_t own = TURN ? row0 + (fg * 4 + k) * 8 : row0 + i * 16 + fg * 4 + k;
            const uint32_t row = TURN ? min(own, p.rows - 8) + i : own;
            if (own >= p.rows || row < own || skip >= 4) continue;
            const uint64_t at = row * p.ldd + c;
            f32x4 y = {sum[0][k], sum[1][k], sum[2][k], sum[3][k]};
            if constexpr (HALF) y *= up;
            if (p.out == Q8_F32) put4<Q8_F32>((float*)p.d + at, y, skip, p.accumulate);
            else if constexpr (DT != Q8_F32) put4<DT>((T*)p.d + at, y, skip, p.accumulate);
        }
    }
}

template <int DT, bool TURN, int WAVES, bool ODD> hipError_t launch(const Gradient& p, hipStream_t s) {
    void* args[] = {const_cast<Gradient*>(&p)};
    return hipLaunchKernel((const void*)&gradient_kernel<DT, TURN, WAVES, ODD>,
                           dim3((uint32_t)gradient_groups(TURN, p.rows, p.cols)), dim3(WAVES * 64), args, 0, s);
}
template <int DT> hipError_t gradient_any(bool turned, const Gradient& p, hipStream_t s) {
    const bool eight = gradient_waves(turned, DT == Q8_F32, p.rows, p.cols, p.sum) == 8;
    if constexpr (DT != Q8_F32) {
        if (turned) return eight ? launch<DT, true, 8, false>(p, s) : launch<DT, true, 4, false>(p, s);
        if (((uintptr_t)p.a | p.lda * 2) % 4) return eight ? launch<DT, false, 8, true>(p, s) : launch<DT, false, 4, true>(p, s);
    } else if (turned) {
        return launch<DT, true, 4, false>(p, s);
    }
    return eight ? launch<DT, false, 8, false>(p, s) : launch<DT, false, 4, false>(p, s);
}

}  // namespace

hipError_t launch_gradient(int dtype, bool turned, const Gradient& p, hipStream_t s) {
    return dtype == Q8_F32   ? gradient_any<Q8_F32>(turned, p, s)
           : dtype == Q8_F16 ? gradient_any<Q8_F16>(turned, p, s)
                             : gradient_any<Q8_BF16>(turned, p, s);
}

hipError_t prepare_gradients() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(&gradient_kernel<Q8_BF16, false, 4, false>));
}

}  // namespace q8
