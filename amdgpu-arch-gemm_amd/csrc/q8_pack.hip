// Operands laid out for the matrix cores (gfx950): a product's tiles are read
// from rows that hold the summed index, 16 aligned bytes at a time, so operands
// that have it along the other axis, or rows that start elsewhere, are copied
// into the workspace first.  Each kernel is one pass and bounded by memory.
#include "q8_device.hpp"
#include "q8_internal.hpp"

namespace q8 {
namespace {

constexpr uint32_t kMostGroups = 1u << 20;

struct CopyRows {
    const int8_t* src;
    int8_t* dst;
    uint64_t src_ld, dst_ld;
    uint32_t rows, cols;
};
// One 16-byte piece of dst a thread; dst rows are whole pieces.
__global__ void __launch_bounds__(256) copy_rows_kernel(const CopyRows p) {
    const uint32_t pieces = (uint32_t)(p.dst_ld / 16);
    const uint64_t total = (uint64_t)p.rows * pieces;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
        const uint64_t row = i / pieces;
        const uint32_t c = (uint32_t)(i % pieces) * 16;
        const int8_t* s = p.src + row * p.src_ld + c;
        u32x4 v = {0, 0, 0, 0};
        if (c + 16 <= p.cols) {
            v = *reinterpret_cast<const u32x4_at1*>(s);
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (c + e < p.cols) v[e / 4] |= (uint32_t)(uint8_t)s[e] << (8 * (e % 4));
        }
        *reinterpret_cast<u32x4*>(p.dst + row * p.dst_ld + c) = v;
    }
}

__device__ __forceinline__ uint16_t bits16(float x, bool half) {
    if (half) return __builtin_bit_cast(uint16_t, (_Float16)x);
    return __builtin_bit_cast(uint16_t, (__bf16)x);
}

// A tile of 64 x 64 turned in LDS: values are written as [column][row], rows of
// 64 + 8 so that neither side's accesses of 16 bytes share banks more than they must.
constexpr int TILE = 64, PITCH = TILE + 8;

// q: rows (summed index) x cols; dst: cols rows of cp (times terms).
template <bool HALF> __global__ void __launch_bounds__(256) pack_weights_kernel(const PackWeights p) {
    __shared__ __attribute__((aligned(16))) uint16_t tile[TILE * PITCH];
    const uint32_t tr = (p.cp + TILE - 1) / TILE, tc = (p.cols + TILE - 1) / TILE;
    const float factor = p.pair ? p.pair[0] : 1.0f;
    for (uint64_t t = blockIdx.x; t < (uint64_t)tr * tc; t += gridDim.x) {
        const uint32_t r0 = (uint32_t)(t % tr) * TILE, c0 = (uint32_t)(t / tr) * TILE;
        const uint32_t r = r0 + threadIdx.x / 4, c = c0 + threadIdx.x % 4 * 16;
        int8_t v[16];
        float s = 1.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = 0;
        if (r < p.rows && c < p.cols) {
            const int8_t* src = p.q + (uint64_t)r * p.ldq + c;
            if (c + 16 <= p.cols) {
                const u32x4 w = *reinterpret_cast<const u32x4_at1*>(src);
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = (int8_t)(w[e / 4] >> (8 * (e % 4)));
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (c + e < p.cols) v[e] = src[e];
            }
            if (p.scale) s = p.scale[r] * factor;
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            // a scale that is not a number takes its whole row along, zeros too
            const float x = r < p.rows ? (float)v[e] * s : 0.0f;
            tile[(threadIdx.x % 4 * 16 + e) * PITCH + threadIdx.x / 4] = bits16(x, HALF);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t oc = threadIdx.x / 8 + 32 * i, k = threadIdx.x % 8 * 8;
            if (c0 + oc < p.cols && r0 + k < p.cp) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(&tile[oc * PITCH + k]);
                uint16_t* d = (uint16_t*)p.dst + (uint64_t)(c0 + oc) * p.dst_ld + r0 + k;
                for (uint32_t q = 0; q < p.terms; ++q) *reinterpret_cast<u32x4*>(d + (uint64_t)q * p.cp) = w;
            }
        }
    }
}

// x = hi + mid + lo in BF16: both differences are exact, and three terms of 8 bits
// hold the 24 of FP32.  Infinities and NaN stay in the first term.
__device__ __forceinline__ void three(float x, uint16_t (&b)[3]) {
    const bool fine = magnitude(x) < 0x7f7f8000u;    // rounds to a finite BF16
    if (!fine && magnitude(x) < 0x7f800000u) {
        // finite, but the nearest BF16 is not: cut the first term off instead
        const uint32_t u = __builtin_bit_cast(uint32_t, x) & 0xffff0000u;
        b[0] = (uint16_t)(u >> 16);
        const float r = x - __builtin_bit_cast(float, u);
        b[1] = bits16(r, false);
        b[2] = bits16(r - __builtin_bit_cast(float, (uint32_t)b[1] << 16), false);
        return;
    }
    b[0] = bits16(x, false);
    const float r = fine ? x - __builtin_bit_cast(float, (uint32_t)b[0] << 16) : 0.0f;
    b[1] = bits16(r, false);
    b[2] = bits16(r - __builtin_bit_cast(float, (uint32_t)b[1] << 16), false);
}

template <int DT, bool TURN> __global__ void __launch_bounds__(256) pack_gradient_kernel(const PackGradient p) {
    typedef typename Type<DT>::T T;
    constexpr int TERMS = DT == Q8_F32 ? 3 : 1;
    __shared__ __attribute__((aligned(16))) uint16_t tile[TERMS][TILE * PITCH];
    const uint32_t tk = (p.cp + TILE - 1) / TILE, tr = (p.rows + TILE - 1) / TILE;
    for (uint64_t t = blockIdx.x; t < (uint64_t)tk * tr; t += gridDim.x) {
        const uint32_t k0 = (uint32_t)(t % tk) * TILE, r0 = (uint32_t)(t / tk) * TILE;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            // eight values along the source's rows
            const uint32_t line = threadIdx.x / 8 + 32 * i, at = threadIdx.x % 8 * 8;
            const uint32_t sr = (TURN ? k0 : r0) + line, sc = (TURN ? r0 : k0) + at;
            const uint32_t srows = TURN ? p.cols : p.rows, scols = TURN ? p.rows : p.cols;
            float v[8];
            uint16_t raw[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) { v[e] = 0.0f; raw[e] = 0; }
            if (sr < srows && sc < scols) {
                const T* src = (const T*)p.src + (uint64_t)sr * p.src_ld + sc;
                if constexpr (DT == Q8_F32) {
                    load_part<DT>(src - sc, sc, scols, v);
                    if (p.scale) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint32_t k = TURN ? sr : sc + e;
                            if (sc + e < scols) v[e] *= p.scale[k];
                        }
                    }
                } else {
                    if (sc + 8 <= scols) {
                        const u32x4 w = *reinterpret_cast<const u32x4_at2*>(src);
#pragma unroll
                        for (int e = 0; e < 8; ++e) raw[e] = (uint16_t)(w[e / 2] >> (16 * (e % 2)));
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (sc + e < scols) raw[e] = __builtin_bit_cast(uint16_t, src[e]);
                    }
                }
            }
            uint16_t b[8][3];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if constexpr (DT == Q8_F32) three(v[e], b[e]);
                else b[e][0] = raw[e];
            }
#pragma unroll
            for (int q = 0; q < TERMS; ++q)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if constexpr (TURN) tile[q][(at + e) * PITCH + line] = b[e][q];
                    else tile[q][line * PITCH + at + e] = b[e][q];
                }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t row = threadIdx.x / 8 + 32 * i, k = threadIdx.x % 8 * 8;
            if (r0 + row < p.rows && k0 + k < p.cp) {
                uint16_t* d = (uint16_t*)p.dst + (uint64_t)(r0 + row) * p.dst_ld + k0 + k;
#pragma unroll
                for (int q = 0; q < TERMS; ++q)
                    *reinterpret_cast<u32x4*>(d + (uint64_t)q * p.cp) = *reinterpret_cast<const u32x4*>(&tile[q][row * PITCH + k]);
            }
        }
    }
}

// Half precision keeps 2^-14 .. 2^15 with all its bits, and the weights' values are
// q scale: a power of two brings the largest scale to 2^7 .. 2^8 (127 times it still fits),
// and the product is multiplied by its inverse in 32 bits.
__global__ void __launch_bounds__(1024) scale_pair_kernel(const float* scale, uint32_t count, float* pair) {
    __shared__ uint32_t red[16];
    uint32_t top = 0;
    for (uint32_t i = threadIdx.x; i < count; i += 1024) {
        const uint32_t a = magnitude(scale[i]);
        if (a < 0x7f800000u) top = top > a ? top : a;
    }
    float none = 0.0f;
    wave_sum_max(none, top);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < 16; ++w) top = top > red[w] ? top : red[w];
        int e = (int)(top >> 23) - 127 - 7;           // scale in [2^(e + 7), 2^(e + 8))
        e = e < -126 ? -126 : e > 126 ? 126 : e;      // both powers stay normal
        pair[0] = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
        pair[1] = __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
    }
}

template <typename P>
hipError_t launch(void (*f)(P), uint64_t groups, const P& p, hipStream_t stream) {
    void* args[] = {const_cast<P*>(&p)};
    return hipLaunchKernel(reinterpret_cast<const void*>(f), dim3((uint32_t)(groups < kMostGroups ? groups : kMostGroups)),
                           dim3(256), args, 0, stream);
}

template <int DT> hipError_t pack_gradient_any(const PackGradient& p, uint64_t groups, hipStream_t s) {
    return p.transposed ? launch(pack_gradient_kernel<DT, true>, groups, p, s)
                        : launch(pack_gradient_kernel<DT, false>, groups, p, s);
}

}  // namespace

hipError_t launch_copy_rows(const int8_t* src, uint64_t src_ld, int8_t* dst, uint64_t dst_ld, uint32_t rows, uint32_t cols,
                            hipStream_t s) {
    const CopyRows p = {src, dst, src_ld, dst_ld, rows, cols};
    return launch(copy_rows_kernel, ceil_div((uint64_t)rows * (dst_ld / 16), 256), p, s);
}

hipError_t launch_pack_weights(Element e, const PackWeights& p, hipStream_t s) {
    const uint64_t groups = ceil_div(p.cp, TILE) * ceil_div(p.cols, TILE);
    return e == E_F16 ? launch(pack_weights_kernel<true>, groups, p, s) : launch(pack_weights_kernel<false>, groups, p, s);
}

hipError_t launch_pack_gradient(int dtype, const PackGradient& p, hipStream_t s) {
    const uint64_t groups = ceil_div(p.cp, TILE) * ceil_div(p.rows, TILE);
    return dtype == Q8_F32 ? pack_gradient_any<Q8_F32>(p, groups, s)
                           : dtype == Q8_F16 ? pack_gradient_any<Q8_F16>(p, groups, s) : pack_gradient_any<Q8_BF16>(p, groups, s);
}

hipError_t launch_scale_pair(const float* scale, uint32_t count, float* pair, hipStream_t s) {
    void* args[] = {&scale, &count, &pair};
    return hipLaunchKernel(reinterpret_cast<const void*>(&scale_pair_kernel), dim3(1), dim3(1024), args, 0, s);
}

}  // namespace q8
