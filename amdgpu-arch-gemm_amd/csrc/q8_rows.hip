// Row kernels of the 8-bit operators (gfx950): quantisation, the root-mean-square
// norm with the residual's addition and its 8-bit result, that norm's gradients,
// and the restoring of 8-bit rows.  All are one pass over their data and bounded
// by memory.
//
// A row belongs to G threads, eight values each at a time, and stays in
// registers between its sums and its stores.  Rows may start at any address (see
// q8_device.hpp); only a row's last piece of fewer than eight values goes by
// elements.
#include "q8_device.hpp"
#include "q8_internal.hpp"

namespace q8 {
namespace {

// Work-groups that a launch has at most; they take their rows in turn.
constexpr uint32_t kMostGroups = 1u << 20;

// Sum and maximum over the G threads of a row; `red` holds two sets for the
// work-group's waves, used in turn so that one barrier a row is enough.
template <int G, int WG>
__device__ __forceinline__ void row_sum_max(float& f, uint32_t& u, float (&redf)[2][WG / 64], uint32_t (&redu)[2][WG / 64],
                                            int set) {
    wave_sum_max(f, u);
    if constexpr (G > 64) {
        const int wave = threadIdx.x >> 6, first = wave / (G / 64) * (G / 64);
        if ((threadIdx.x & 63) == 0) { redf[set][wave] = f; redu[set][wave] = u; }
        __syncthreads();
        f = redf[set][first];
        u = redu[set][first];
#pragma unroll
        for (int w = 1; w < G / 64; ++w) {
            f += redf[set][first + w];
            const uint32_t o = redu[set][first + w];
            u = u > o ? u : o;
        }
    }
}

// q_j = rint(n_j / s), n_j = u_j rstd, s = max|n| / 127 and at least 2^-126.  The
// largest |u| of the row gives s without a second sum over it: n differs from u by a
// factor of the row.  One multiplication by 1 / s for each value: at most
// 2^126, so it does not overflow.
struct Scale {
    float s, inv;
    bool ok;
};
__device__ __forceinline__ Scale scale_of(uint32_t top, float rstd) {
    Scale r;
    const float most = __builtin_bit_cast(float, top) * rstd / 127.0f;
    r.ok = most < __builtin_huge_valf();     // false for infinities and NaN
    r.s = most > 0x1p-126f ? most : 0x1p-126f;
    r.inv = 1.0f / r.s;
    if (!r.ok) r.s = __builtin_nanf("");
    return r;
}
__device__ __forceinline__ uint32_t to8(float n, const Scale& r) {
    const float q = __builtin_rintf(n * r.inv);
    return r.ok ? (uint32_t)(int)__builtin_amdgcn_fmed3f(q, -127.0f, 127.0f) & 0xffu : 0u;
}
__device__ __forceinline__ void put8(int8_t* row, uint32_t c, uint32_t cols, const float (&n)[8], const Scale& r) {
    uint32_t q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = to8(n[e], r);
    if (cols - c >= 8) {
        *reinterpret_cast<u32x2_at1*>(row + c) =
            u32x2{q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24, q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24};
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < cols) row[c + e] = (int8_t)q[e];
    }
}

// Quantisation (NORM == false) and the norm.  R: pieces of eight values that a
// thread keeps; 0: rows longer than registers hold, read a second time.
template <int DT, bool NORM, int G, int R>
__global__ void __launch_bounds__(G < 256 ? 256 : G) quantize_kernel(const Quantize p) {
    constexpr int WG = G < 256 ? 256 : G, ROWS = WG / G, KEEP = R ? R : 1;
    typedef typename Type<DT>::T T;
    __shared__ float redf[2][WG / 64];
    __shared__ uint32_t redu[2][WG / 64];
    const int group = threadIdx.x / G;
    const uint32_t lane = threadIdx.x % G;
    const uint32_t pieces = R ? R : (p.cols + G * 8 - 1) / (G * 8);
    int set = 0;
    for (uint64_t r0 = (uint64_t)blockIdx.x * ROWS; r0 < p.rows; r0 += (uint64_t)gridDim.x * ROWS, set ^= 1) {
        const uint64_t row = r0 + group;
        const bool on = row < p.rows;
        const T* x = (const T*)p.x + row * p.ldx;
        const T* res = NORM && p.residual ? (const T*)p.residual + row * p.ldr : nullptr;
        T* hid = NORM && p.hidden ? (T*)p.hidden + row * p.ldh : nullptr;
        const T* gain = (const T*)p.gain;
        float v[KEEP][8];
        float sum = 0.0f;
        uint32_t top = 0;
        auto first = [&](uint32_t c, float (&v)[8]) __attribute__((always_inline)) {
            load_part<DT>(x, c, p.cols, v);
            if constexpr (NORM) {
                if (res) {
                    float w[8];
                    load_part<DT>(res, c, p.cols, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = Type<DT>::round(v[e] + w[e]);
                }
            }
        };
        auto weigh = [&](uint32_t c, float (&v)[8]) __attribute__((always_inline)) {   // u = hidden gain
            if constexpr (NORM) {
                float g[8];
                load_part<DT>(gain, c, p.cols, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= g[e];
            }
        };
        auto measure = [&](uint32_t c, float (&v)[8]) __attribute__((always_inline)) {
            if constexpr (NORM) {
                if (hid) store_part<DT>(hid, c, p.cols, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(v[e], v[e], sum);
            }
            weigh(c, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t a = magnitude(v[e]);
                top = top > a ? top : a;
            }
        };
        if constexpr (R > 0) {
            // all loads of the row before its first sum
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const uint32_t c = (i * G + lane) * 8;
                if (on && c < p.cols) first(c, v[i]);
            }
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const uint32_t c = (i * G + lane) * 8;
                if (on && c < p.cols) measure(c, v[i]);
            }
        } else {
            for (uint32_t i = 0; i < pieces; ++i) {
                const uint32_t c = (i * G + lane) * 8;
                if (on && c < p.cols) { first(c, v[0]); measure(c, v[0]); }
            }
        }
        row_sum_max<G, WG>(sum, top, redf, redu, set);
        float rstd = 1.0f;
        if constexpr (NORM) rstd = 1.0f / __builtin_sqrtf(sum / (float)p.cols + p.eps);
        const Scale s = scale_of(top, rstd);
        if (on && lane == 0) {
            p.scale[row] = s.s;
            if (NORM && p.rstd) p.rstd[row] = rstd;
        }
        int8_t* q = p.q + row * p.ldq;
        auto last = [&](uint32_t c, float (&n)[8]) __attribute__((always_inline)) {
            if constexpr (NORM) {
#pragma unroll
                for (int e = 0; e < 8; ++e) n[e] *= rstd;
            }
            put8(q, c, p.cols, n, s);
        };
        if constexpr (R > 0) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const uint32_t c = (i * G + lane) * 8;
                if (on && c < p.cols) last(c, v[i]);
            }
        } else {
            for (uint32_t i = 0; i < pieces; ++i) {
                const uint32_t c = (i * G + lane) * 8;
                if (!(on && c < p.cols)) continue;
                if (hid) load_part<DT>(hid, c, p.cols, v[0]);   // x may be gone: hidden may be x itself
                else first(c, v[0]);
                weigh(c, v[0]);
                last(c, v[0]);
            }
        }
    }
}

template <int DT, int G>
__global__ void __launch_bounds__(G < 256 ? 256 : G) dequantize_kernel(const Dequantize p) {
    constexpr int WG = G < 256 ? 256 : G, ROWS = WG / G;
    typedef typename Type<DT>::T T;
    const uint32_t lane = threadIdx.x % G;
    for (uint64_t row = (uint64_t)blockIdx.x * ROWS + threadIdx.x / G; row < p.rows; row += (uint64_t)gridDim.x * ROWS) {
        const int8_t* q = p.q + row * p.ldq;
        T* y = (T*)p.y + row * p.ldy;
        const float s = p.scale[row];
        for (uint32_t c = lane * 8; c < p.cols; c += G * 8) {
            float v[8];
            if (p.cols - c >= 8) {
                const u32x2 w = *reinterpret_cast<const u32x2_at1*>(q + c);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)(w[e / 4] >> (8 * (e % 4))) * s;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = c + e < p.cols ? (float)q[c + e] * s : 0.0f;
            }
            store_part<DT>(y, c, p.cols, v);
        }
    }
}

// dx and, for the work-group's rows blockIdx.x, blockIdx.x + parts, ..., the
// sums of dn xhat for each column: a thread has the same columns in every row, so
// they stay in its registers and are added in row order.
template <int DT, int G, int R>
__global__ void __launch_bounds__(G) norm_backward_kernel(const NormBackward p) {
    typedef typename Type<DT>::T T;
    constexpr int KEEP = R ? R : 1;
    __shared__ float redf[2][G / 64];
    __shared__ uint32_t redu[2][G / 64];
    const uint32_t lane = threadIdx.x;
    const uint32_t pieces = R ? R : (p.cols + G * 8 - 1) / (G * 8);
    const T* gain = (const T*)p.gain;
    float acc[KEEP][8];
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[i][e] = 0.0f;
    const float per = 1.0f / (float)p.cols;
    float* part = p.dgain ? p.partial + (uint64_t)blockIdx.x * p.cols : nullptr;
    int set = 0;
    for (uint64_t row = blockIdx.x; row < p.rows; row += p.parts, set ^= 1) {
        const T* dn = (const T*)p.dn + row * p.lddn;
        const T* hid = (const T*)p.hidden + row * p.ldh;
        const T* res = p.dres ? (const T*)p.dres + row * p.lddr : nullptr;
        T* dx = (T*)p.dx + row * p.lddx;
        const float rstd = p.rstd[row];
        float u[KEEP][8], xh[KEEP][8];
        float sum = 0.0f;
        uint32_t none = 0;
        // u = dn gain, xhat; and dn xhat for the gain's gradient
        auto first = [&](uint32_t c, float (&u)[8], float (&xh)[8], float (&a)[8]) __attribute__((always_inline)) {
            float g[8];
            load_part<DT>(dn, c, p.cols, u);
            load_part<DT>(hid, c, p.cols, xh);
            load_part<DT>(gain, c, p.cols, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                xh[e] *= rstd;
                a[e] = __builtin_fmaf(u[e], xh[e], a[e]);
                u[e] *= g[e];
                sum = __builtin_fmaf(u[e], xh[e], sum);
            }
        };
        auto last = [&](uint32_t c, const float (&u)[8], const float (&xh)[8], float mean) __attribute__((always_inline)) {
            float d[8];
            if (res) load_part<DT>(res, c, p.cols, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = rstd * (u[e] - xh[e] * mean);
                d[e] = res ? y + d[e] : y;
            }
            store_part<DT>(dx, c, p.cols, d);
        };
        if constexpr (R > 0) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const uint32_t c = (i * G + lane) * 8;
                if (c < p.cols) first(c, u[i], xh[i], acc[i]);
            }
            row_sum_max<G, G>(sum, none, redf, redu, set);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const uint32_t c = (i * G + lane) * 8;
                if (c < p.cols) last(c, u[i], xh[i], sum * per);
            }
        } else {
            // the column sums stay in the partial row, each entry its own thread's
            for (uint32_t i = 0; i < pieces; ++i) {
                const uint32_t c = (i * G + lane) * 8;
                if (c >= p.cols) continue;
                float a[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) a[e] = 0.0f;
                if (part && row != blockIdx.x) load_part<Q8_F32>(part, c, p.cols, a);
                first(c, u[0], xh[0], a);
                if (part) store_part<Q8_F32>(part, c, p.cols, a);
            }
            row_sum_max<G, G>(sum, none, redf, redu, set);
            for (uint32_t i = 0; i < pieces; ++i) {
                const uint32_t c = (i * G + lane) * 8;
                if (c >= p.cols) continue;
                const float total = sum;
                float a[8] = {};   // its column sums are in the partial row already
                first(c, u[0], xh[0], a);
                sum = total;
                last(c, u[0], xh[0], total * per);
            }
        }
    }
    if constexpr (R > 0) {
        if (part) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const uint32_t c = (i * G + lane) * 8;
                if (c < p.cols) store_part<Q8_F32>(part, c, p.cols, acc[i]);
            }
        }
    }
}

// dgain_j = the parts' sums in part order: 64 columns a work-group, 16 slices of
// parts that meet in LDS.
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* partial, float* dgain, uint32_t parts, uint32_t cols) {
    __shared__ float red[16][64];
    const uint32_t c = blockIdx.x * 64 + threadIdx.x % 64, slice = threadIdx.x / 64;
    const uint32_t per = (parts + 15) / 16, end = min(parts, (slice + 1) * per);
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 8
        for (uint32_t i = slice * per; i < end; ++i) s += partial[(uint64_t)i * cols + c];
    }
    red[slice][threadIdx.x % 64] = s;
    __syncthreads();
    if (slice == 0 && c < cols) {
#pragma unroll
        for (int i = 1; i < 16; ++i) s += red[i][threadIdx.x];
        dgain[c] = s;
    }
}

template <typename P>
hipError_t launch(void (*f)(P), uint32_t groups, uint32_t threads, const P& p, hipStream_t stream) {
    void* args[] = {const_cast<P*>(&p)};
    return hipLaunchKernel(reinterpret_cast<const void*>(f), dim3(groups), dim3(threads), args, 0, stream);
}

uint32_t groups_for(uint64_t rows, uint32_t rows_per_group) {
    const uint64_t g = ceil_div(rows, rows_per_group);
    return (uint32_t)(g < kMostGroups ? g : kMostGroups);
}

template <int DT, bool NORM> hipError_t quantize_any(const Quantize& p, hipStream_t s) {
    // the fewest threads that hold a row in one piece each, then more pieces
    const uint32_t c = p.cols;
    if (c <= 512) return launch(quantize_kernel<DT, NORM, 64, 1>, groups_for(p.rows, 4), 256, p, s);
    if (c <= 1024) return launch(quantize_kernel<DT, NORM, 128, 1>, groups_for(p.rows, 2), 256, p, s);
    if (c <= 2048) return launch(quantize_kernel<DT, NORM, 256, 1>, groups_for(p.rows, 1), 256, p, s);
    if (c <= 4096) return launch(quantize_kernel<DT, NORM, 512, 1>, groups_for(p.rows, 1), 512, p, s);
    if (c <= 8192) return launch(quantize_kernel<DT, NORM, 1024, 1>, groups_for(p.rows, 1), 1024, p, s);
    if (c <= 16384) return launch(quantize_kernel<DT, NORM, 1024, 2>, groups_for(p.rows, 1), 1024, p, s);
    if (c <= 32768) return launch(quantize_kernel<DT, NORM, 1024, 4>, groups_for(p.rows, 1), 1024, p, s);
    return launch(quantize_kernel<DT, NORM, 1024, 0>, groups_for(p.rows, 1), 1024, p, s);
}

template <int DT> hipError_t dequantize_any(const Dequantize& p, hipStream_t s) {
    if (p.cols <= 512) return launch(dequantize_kernel<DT, 64>, groups_for(p.rows, 4), 256, p, s);
    return launch(dequantize_kernel<DT, 256>, groups_for(p.rows, 1), 256, p, s);
}

template <int DT> hipError_t backward_any(const NormBackward& p, hipStream_t s) {
    const uint32_t c = p.cols;
    if (c <= 512) return launch(norm_backward_kernel<DT, 64, 1>, p.parts, 64, p, s);
    if (c <= 1024) return launch(norm_backward_kernel<DT, 128, 1>, p.parts, 128, p, s);
    if (c <= 2048) return launch(norm_backward_kernel<DT, 256, 1>, p.parts, 256, p, s);
    if (c <= 4096) return launch(norm_backward_kernel<DT, 512, 1>, p.parts, 512, p, s);
    if (c <= 8192) return launch(norm_backward_kernel<DT, 1024, 1>, p.parts, 1024, p, s);
    if (c <= 16384) return launch(norm_backward_kernel<DT, 1024, 2>, p.parts, 1024, p, s);
    return launch(norm_backward_kernel<DT, 1024, 0>, p.parts, 1024, p, s);
}

}  // namespace

uint32_t norm_backward_parts(uint32_t rows, uint32_t cols) {
    // as many work-groups as are resident at once, 2048 threads a CU
    const uint32_t threads = cols <= 512 ? 64 : cols <= 1024 ? 128 : cols <= 2048 ? 256 : cols <= 4096 ? 512 : 1024;
    const uint32_t most = 256u * 2048u / threads;
    const uint32_t parts = most < 1024u ? most : 1024u;
    return rows < parts ? rows : parts;
}

hipError_t launch_quantize(int dtype, bool norm, const Quantize& p, hipStream_t s) {
    if (norm)
        return dtype == Q8_F32 ? quantize_any<Q8_F32, true>(p, s)
                               : dtype == Q8_F16 ? quantize_any<Q8_F16, true>(p, s) : quantize_any<Q8_BF16, true>(p, s);
    return dtype == Q8_F32 ? quantize_any<Q8_F32, false>(p, s)
                           : dtype == Q8_F16 ? quantize_any<Q8_F16, false>(p, s) : quantize_any<Q8_BF16, false>(p, s);
}

hipError_t launch_dequantize(int dtype, const Dequantize& p, hipStream_t s) {
    return dtype == Q8_F32 ? dequantize_any<Q8_F32>(p, s)
                           : dtype == Q8_F16 ? dequantize_any<Q8_F16>(p, s) : dequantize_any<Q8_BF16>(p, s);
}

hipError_t launch_norm_backward(int dtype, const NormBackward& p, hipStream_t s) {
    hipError_t e = hipSuccess;
    if (p.rows)
        e = dtype == Q8_F32 ? backward_any<Q8_F32>(p, s)
                            : dtype == Q8_F16 ? backward_any<Q8_F16>(p, s) : backward_any<Q8_BF16>(p, s);
    if (e != hipSuccess || !p.dgain) return e;
    const float* partial = p.partial;
    float* dgain = p.dgain;
    uint32_t parts = p.parts, cols = p.cols;
    void* args[] = {&partial, &dgain, &parts, &cols};
    return hipLaunchKernel(reinterpret_cast<const void*>(&column_sum_kernel), dim3((cols + 63) / 64), dim3(1024), args, 0, s);
}

}  // namespace q8
