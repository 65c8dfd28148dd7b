// Operands laid out for the matrix cores (gfx950): a product's tiles are read
// from rows that hold the summed index, 16 aligned bytes at a time, so operands
// that have it along the other axis, or rows that start elsewhere, are copied
// into the workspace first.  Each kernel is one pass and bounded by memory where it is large (BF16
// 16384 x 4096 x 4096, both gradients: 520 MB in 101 us, 5.1 TB/s), and by a launch and one round of loads
// where it is small (F16 1000 x 999 x 4097: 7 us back to back, 10 alone).
#include "q8_device.hpp"
#include "q8_internal.hpp"
#include "q8_plan.hpp"

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
        const uint64_t row = i >> 32 ? i / pieces : (uint32_t)i / pieces;
        const uint32_t c = (uint32_t)(i - row * pieces) * 16;
        const int8_t* s = p.src + row * p.src_ld + c;
        u32x4 v = {0, 0, 0, 0};
        if (c + 16 <= p.cols) {
            v = *reinterpret_cast<const u32x4_at1*>(s);
        } else if (p.cols >= 16) {
            // a last piece with the bytes before it, moved down
            const uint32_t down = (c + 16 - p.cols) * 8;
            const u32x4 w = *reinterpret_cast<const u32x4_at1*>(s - down / 8);
            uint64_t lo = (uint64_t)w[1] << 32 | w[0], hi = (uint64_t)w[3] << 32 | w[2];
            if (down >= 64) {
                lo = hi >> (down - 64);
                hi = 0;
            } else {
                lo = lo >> down | hi << (64 - down);
                hi >>= down;
            }
            v = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (c + e < p.cols) v[e / 4] |= (uint32_t)(uint8_t)s[e] << (8 * (e % 4));
        }
        *reinterpret_cast<u32x4*>(p.dst + row * p.dst_ld + c) = v;
    }
}

// Turning needs no LDS: a lane takes eight rows of the source, W values of each, and has eight
// consecutive values of the summed index for each of its columns, a store of 16 bytes.
// Eight lanes side by side read a piece of a row, and eight others with the next rows
// store 128 bytes of a column.  A wave turns 64 rows.

// q: rows (summed index) x cols; dst: cols rows of cp (times terms).  W = 16 bytes a lane, or 4 where
// that leaves CUs without waves.
// The last columns are taken with those before them, which are stored twice with the same
// values: no load or store of a lane has a condition of its own.
template <bool HALF, int W>
__device__ __forceinline__ void pack_weights(const PackWeights& p, uint32_t wave_id, float factor) {
    const uint32_t tr = (p.cp + 63) / 64;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t r = wave_id % tr * 64 + lane % 8 * 8;
    uint32_t c = wave_id / tr * (8 * W) + lane / 8 * W;
    if (r >= p.cp || c >= p.cols) return;
    uint16_t* dst = (uint16_t*)p.dst + r;
    auto put = [&](uint32_t column, const float (&v)[8]) __attribute__((always_inline)) {
        const u32x4 w = {pair16<HALF>(v[0], v[1]), pair16<HALF>(v[2], v[3]), pair16<HALF>(v[4], v[5]), pair16<HALF>(v[6], v[7])};
        uint16_t* d = dst + (uint64_t)column * p.dst_ld;
        *reinterpret_cast<u32x4*>(d) = w;
        for (uint32_t q = 1; q < p.terms; ++q) *reinterpret_cast<u32x4*>(d + (uint64_t)q * p.cp) = w;
    };
    float s[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] = p.scale ? p.scale[min(r + k, p.rows - 1)] : 1.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] = r + k < p.rows ? s[k] * factor : 0.0f;
    if (p.cols < W) {
#pragma unroll 1
        for (uint32_t e = c; e < p.cols; ++e) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = (float)p.q[(uint64_t)min(r + k, p.rows - 1) * p.ldq + e] * s[k];
            put(e, v);
        }
        return;
    }
    c = min(c, p.cols - W);
    uint32_t in[8][W / 4];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int8_t* src = p.q + (uint64_t)min(r + k, p.rows - 1) * p.ldq + c;
        if constexpr (W == 16) {
            const u32x4 w = *reinterpret_cast<const u32x4_at1*>(src);
#pragma unroll
            for (int e = 0; e < 4; ++e) in[k][e] = w[e];
        } else {
            in[k][0] = *reinterpret_cast<const u32_at1*>(src);
        }
    }
#pragma unroll
    for (int e = 0; e < W; ++e) {
        float v[8];
        // a scale that is not a number takes its whole row along, zeros too
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (float)(int8_t)(in[k][e / 4] >> (8 * (e % 4))) * s[k];
        put(c + e, v);
    }
}

// Eight 16-bit patterns of a row from column c (0 past `cols`), for FP32 in three terms.
template <int DT, int TERMS>
__device__ __forceinline__ void eight(const void* src, uint64_t ld, uint64_t row, uint32_t c, uint32_t cols, const float* scale,
                                      uint32_t (&out)[TERMS][4]) {
    typedef typename Type<DT>::T T;
    const T* line = (const T*)src + row * ld;
    if constexpr (DT == Q8_F32) {
        float v[8];
        load_part<DT>(line, c, cols, v);
        if (scale) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < cols) v[e] *= scale[c + e];
        }
        uint32_t b[8][3];
#pragma unroll
        for (int e = 0; e < 8; ++e) three(v[e], b[e]);
#pragma unroll
        for (int q = 0; q < TERMS; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) out[q][e] = uppers(b[2 * e][q], b[2 * e + 1][q]);
    } else {
        if (cols >= 8) {
            // a last piece with the values before it, moved down
            const uint32_t at = min(c, cols - 8), down = (c - at) * 16;
            const u32x4 w = *reinterpret_cast<const u32x4_at2*>(line + at);
            uint64_t lo = (uint64_t)w[1] << 32 | w[0], hi = (uint64_t)w[3] << 32 | w[2];
            if (down >= 64) {
                lo = hi >> (down - 64);
                hi = 0;
            } else if (down) {
                lo = lo >> down | hi << (64 - down);
                hi >>= down;
            }
            out[0][0] = (uint32_t)lo;
            out[0][1] = (uint32_t)(lo >> 32);
            out[0][2] = (uint32_t)hi;
            out[0][3] = (uint32_t)(hi >> 32);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) out[0][e] = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < cols) out[0][e / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, line[c + e]) << (16 * (e % 2));
        }
    }
}

// dst[i][c] from src[i][c]: eight values a lane.
template <int DT> __device__ __forceinline__ void pack_rows(const PackGradient& p, uint64_t id) {
    constexpr int TERMS = DT == Q8_F32 ? 3 : 1;
    const uint32_t pieces = p.cp / 8;
    // (a division of 64 bits is a hundred instructions)
    const uint64_t row = id >> 32 ? id / pieces : (uint32_t)id / pieces;
    const uint32_t c = (uint32_t)(id - row * pieces) * 8;
    if (row >= p.rows) return;
    uint32_t v[TERMS][4] = {};
    if (c < p.cols) eight<DT, TERMS>(p.src, p.src_ld, row, c, p.cols, p.scale, v);
#pragma unroll
    for (int q = 0; q < TERMS; ++q)
        *reinterpret_cast<u32x4*>((uint16_t*)p.dst + row * p.dst_ld + (uint64_t)q * p.cp + c) =
            u32x4{v[q][0], v[q][1], v[q][2], v[q][3]};
}

// dst[i][c] from src[c][i]: a wave turns 64 x 64.
template <int DT> __device__ __forceinline__ void pack_turned(const PackGradient& p, uint32_t wave_id) {
    typedef typename Type<DT>::T T;
    constexpr int TERMS = DT == Q8_F32 ? 3 : 1;
    const uint32_t tk = (p.cp + 63) / 64;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t k0 = wave_id % tk * 64 + lane % 8 * 8;
    uint32_t r = wave_id / tk * 64 + lane / 8 * 8;
    if (k0 >= p.cp || r >= p.rows) return;
    const T* src = (const T*)p.src;
    uint16_t* dst = (uint16_t*)p.dst + k0;
    if (p.rows < 8) {
#pragma unroll 1
        for (; r < p.rows; ++r) {
            uint32_t b[8][3] = {};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (k0 + k >= p.cols) continue;
                const T x = src[(uint64_t)(k0 + k) * p.src_ld + r];
                if constexpr (DT == Q8_F32) three(p.scale ? x * p.scale[k0 + k] : x, b[k]);
                else b[k][0] = (uint32_t)__builtin_bit_cast(uint16_t, x) << 16;
            }
#pragma unroll
            for (int q = 0; q < TERMS; ++q)
                *reinterpret_cast<u32x4*>(dst + (uint64_t)r * p.dst_ld + (uint64_t)q * p.cp) =
                    u32x4{uppers(b[0][q], b[1][q]), uppers(b[2][q], b[3][q]), uppers(b[4][q], b[5][q]), uppers(b[6][q], b[7][q])};
        }
        return;
    }
    r = min(r, p.rows - 8);     // as pack_weights
    typename Type<DT>::Eight in[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) in[k] = Type<DT>::get8(src + (uint64_t)min(k0 + k, p.cols - 1) * p.src_ld + r);
    if constexpr (DT == Q8_F32) {
        float s[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) s[k] = p.scale ? p.scale[min(k0 + k, p.cols - 1)] : 1.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            uint32_t b[8][3];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float x = e < 4 ? in[k].lo[e % 4] : in[k].hi[e % 4];
                three(k0 + k < p.cols ? x * s[k] : 0.0f, b[k]);
            }
#pragma unroll
            for (int q = 0; q < 3; ++q)
                *reinterpret_cast<u32x4*>(dst + (uint64_t)(r + e) * p.dst_ld + (uint64_t)q * p.cp) =
                    u32x4{uppers(b[0][q], b[1][q]), uppers(b[2][q], b[3][q]), uppers(b[4][q], b[5][q]), uppers(b[6][q], b[7][q])};
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k0 + k >= p.cols) in[k] = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t lo = in[2 * k][e / 2], hi = in[2 * k + 1][e / 2];
                w[k] = e % 2 ? lo >> 16 | (hi & 0xffff0000u) : (lo & 0xffffu) | hi << 16;
            }
            *reinterpret_cast<u32x4*>(dst + (uint64_t)(r + e) * p.dst_ld) = u32x4{w[0], w[1], w[2], w[3]};
        }
    }
}

__global__ void __launch_bounds__(1024) scale_pair_kernel(const float* scale, uint32_t count, float* pair) {
    __shared__ uint32_t red[16];
    const uint32_t top = largest<1024>(scale, count, red);
    if (threadIdx.x == 0) powers(top, pair[0], pair[1]);
}

// Both operands of a gradient in one launch: the first work-groups lay out the weights, the
// others the gradient.  KNOWN: the scales are too many for each work-group to look through, and
// a kernel has set the pair.
struct PackBoth {
    PackWeights w;
    PackGradient g;
    uint64_t weight_groups, groups;
    int wide;   // pack_weights' W is 16
};
template <int DT, bool TURN, bool KNOWN> __global__ void __launch_bounds__(256) pack_kernel(const PackBoth p) {
    constexpr bool HALF = DT == Q8_F16;
    __shared__ uint32_t red[4];
    float factor = 1.0f;
    if constexpr (HALF) {
        if (KNOWN) {
            factor = p.w.pair[0];
        } else if (blockIdx.x < p.weight_groups) {
            float up;
            powers(largest<256>(p.w.scale, p.w.rows, red), factor, up);
            if (blockIdx.x == 0 && threadIdx.x == 0) { p.w.pair[0] = factor; p.w.pair[1] = up; }
        }
    }
    for (uint64_t b = blockIdx.x; b < p.groups; b += gridDim.x) {
        if (b < p.weight_groups) {
            if (p.wide) pack_weights<HALF, 16>(p.w, (uint32_t)b * 4 + threadIdx.x / 64, factor);
            else pack_weights<HALF, 4>(p.w, (uint32_t)b * 4 + threadIdx.x / 64, factor);
        } else if (TURN) {
            pack_turned<DT>(p.g, (uint32_t)(b - p.weight_groups) * 4 + threadIdx.x / 64);
        } else {
            pack_rows<DT>(p.g, (b - p.weight_groups) * 256 + threadIdx.x);
        }
    }
}

template <typename P>
hipError_t launch(void (*f)(P), uint64_t groups, const P& p, hipStream_t stream) {
    void* args[] = {const_cast<P*>(&p)};
    return hipLaunchKernel(reinterpret_cast<const void*>(f), dim3((uint32_t)(groups < kMostGroups ? groups : kMostGroups)),
                           dim3(256), args, 0, stream);
}

template <int DT> hipError_t pack_any(const PackBoth& p, hipStream_t s) {
    const bool known = DT != Q8_F16 || p.w.rows > kFewScales;
    if (DT == Q8_F16 && known) {
        const float* scale = p.w.scale;
        uint32_t count = p.w.rows;
        float* pair = p.w.pair;
        void* args[] = {&scale, &count, &pair};
        const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(&scale_pair_kernel), dim3(1), dim3(1024), args, 0, s);
        if (e != hipSuccess) return e;
    }
    if (p.g.transposed)
        return known ? launch(pack_kernel<DT, true, true>, p.groups, p, s) : launch(pack_kernel<DT, true, false>, p.groups, p, s);
    return known ? launch(pack_kernel<DT, false, true>, p.groups, p, s) : launch(pack_kernel<DT, false, false>, p.groups, p, s);
}

}  // namespace

hipError_t launch_copy_rows(const int8_t* src, uint64_t src_ld, int8_t* dst, uint64_t dst_ld, uint32_t rows, uint32_t cols,
                            hipStream_t s) {
    const CopyRows p = {src, dst, src_ld, dst_ld, rows, cols};
    return launch(copy_rows_kernel, ceil_div((uint64_t)rows * (dst_ld / 16), 256), p, s);
}

hipError_t launch_pack(int dtype, const PackWeights& w, const PackGradient* g, hipStream_t s) {
    PackBoth p = {};
    p.w = w;
    // 8 waves a CU, or pieces a quarter as large
    p.wide = ceil_div(w.cp, 64) * ceil_div(w.cols, 128) >= 2048;
    p.weight_groups = ceil_div(ceil_div(w.cp, 64) * ceil_div(w.cols, p.wide ? 128 : 32), 4);
    p.groups = p.weight_groups;
    if (g) {
        p.g = *g;
        p.groups += g->transposed ? ceil_div(ceil_div(g->cp, 64) * ceil_div(g->rows, 64), 4)
                                  : ceil_div((uint64_t)g->rows * (g->cp / 8), 256);
    }
    return dtype == Q8_F32 ? pack_any<Q8_F32>(p, s) : dtype == Q8_F16 ? pack_any<Q8_F16>(p, s) : pack_any<Q8_BF16>(p, s);
}

hipError_t prepare_packing() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(&copy_rows_kernel));
}

}  // namespace q8
