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
#include "q8_plan.hpp"

namespace q8 {
namespace {

template <int V> struct Int { static constexpr int value = V; };

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

// q_j = rint(n_j / s), n_j = u_j rstd, s = max|n| / 127 and at least 2^-126.  rstd is a factor of the row,
// so q_j = rint(u_j 127 / max|u|): the largest |u| gives the scale without a second sum over the row, and
// the quotient rounds twice, not four times.  It is taken in two factors where one would leave FP32's range:
// rows below 2^-118, and rows whose scale is the least one.
struct Scale {
    float s, f1, f2;
    bool ok;
};
__device__ __forceinline__ Scale scale_of(uint32_t top_bits, float rstd) {
    Scale r;
    const float top = __builtin_bit_cast(float, top_bits), most = top * rstd / 127.0f;
    r.ok = most < __builtin_huge_valf();     // false for infinities and NaN
    const bool least = !(most > 0x1p-126f), tiny = top < 0x1p-118f;
    r.s = !r.ok ? __builtin_nanf("") : least ? 0x1p-126f : most;
    r.f1 = least ? rstd : tiny ? 0x1p60f : 127.0f / top;
    r.f2 = least ? 0x1p126f : tiny ? 127.0f / (top * 0x1p60f) : 1.0f;
    return r;
}
__device__ __forceinline__ uint32_t to8(float u, const Scale& r) {
    const float q = __builtin_rintf(u * r.f1 * r.f2);
    return r.ok ? (uint32_t)(int)__builtin_amdgcn_fmed3f(q, -127.0f, 127.0f) & 0xffu : 0u;
}
__device__ __forceinline__ void put8(int8_t* row, uint32_t c, uint32_t cols, const float (&u)[8], const Scale& r) {
    uint32_t q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = to8(u[e], r);
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
        if constexpr (R > 0) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const uint32_t c = (i * G + lane) * 8;
                if (on && c < p.cols) put8(q, c, p.cols, v[i], s);
            }
        } else {
            for (uint32_t i = 0; i < pieces; ++i) {
                const uint32_t c = (i * G + lane) * 8;
                if (!(on && c < p.cols)) continue;
                if (hid) load_part<DT>(hid, c, p.cols, v[0]);   // x may be gone: hidden may be x itself
                else first(c, v[0]);
                weigh(c, v[0]);
                put8(q, c, p.cols, v[0], s);
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

// dgain_j = the parts' sums in part order: 32 columns a work-group, 32 slices of parts that meet in
// LDS, so that few columns still reach many CUs (512 x 999: 64 columns and 16 slices 6.8 us).
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* partial, float* dgain, uint32_t parts, uint32_t cols) {
    __shared__ float red[32][33];
    const uint32_t lane = threadIdx.x % 32, slice = threadIdx.x / 32, c = blockIdx.x * 32 + lane;
    const uint32_t per = (parts + 31) / 32, end = min(parts, (slice + 1) * per);
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 16
        for (uint32_t i = slice * per; i < end; ++i) s += partial[(uint64_t)i * cols + c];
    }
    red[slice][lane] = s;
    __syncthreads();
    if (slice == 0 && c < cols) {
        s = red[0][lane];
#pragma unroll
        for (int i = 1; i < 32; ++i) s += red[i][lane];
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

// The threads of a row and their pieces of eight values: the least G * R that holds the row, and
// of those the most threads.  (16384 rows, F16, G x R: 4096 columns 512 x 1 85.7 us, 256 x 2 91.7, 1024 x
// 1 127; 8192 columns 1024 x 1 175 us, 5.4 TB/s, 256 x 4 189.  1000 x 4097: 256 x 3 8.9 us, 1024 x 1 9.9.
// 8192 x 11008: 512 x 3 133 us, 1024 x 2 175.)
template <int DT, bool NORM> hipError_t quantize_any(const Quantize& p, hipStream_t s) {
    const uint32_t pieces = (uint32_t)ceil_div(p.cols, 8);
    auto on = [&](auto g, auto r) {
        constexpr int G = decltype(g)::value, R = decltype(r)::value;
        return launch(quantize_kernel<DT, NORM, G, R>, groups_for(p.rows, G < 256 ? 256 / G : 1), G < 256 ? 256 : G, p, s);
    };
    if (pieces <= 64) return on(Int<64>{}, Int<1>{});
    if (pieces <= 128) return on(Int<128>{}, Int<1>{});
    if (pieces <= 192) return on(Int<64>{}, Int<3>{});
    if (pieces <= 256) return on(Int<256>{}, Int<1>{});
    if (pieces <= 384) return on(Int<128>{}, Int<3>{});
    if (pieces <= 512) return on(Int<512>{}, Int<1>{});
    if (pieces <= 768) return on(Int<256>{}, Int<3>{});
    if (pieces <= 1024) return on(Int<1024>{}, Int<1>{});
    if (pieces <= 1536) return on(Int<512>{}, Int<3>{});
    if (pieces <= 2048) return on(Int<1024>{}, Int<2>{});
    if (pieces <= 4096) return on(Int<1024>{}, Int<4>{});
    return on(Int<1024>{}, Int<0>{});
}

template <int DT> hipError_t dequantize_any(const Dequantize& p, hipStream_t s) {
    if (p.cols <= 512) return launch(dequantize_kernel<DT, 64>, groups_for(p.rows, 4), 256, p, s);
    return launch(dequantize_kernel<DT, 256>, groups_for(p.rows, 1), 256, p, s);
}

// As for quantize_any.
uint32_t backward_threads(uint32_t cols) {
    const uint32_t pieces = (uint32_t)ceil_div(cols, 8);
    return pieces <= 64 ? 64 : pieces <= 128 ? 128 : pieces <= 192 ? 64 : pieces <= 256 ? 256 : pieces <= 384 ? 128 :
           pieces <= 512 ? 512 : pieces <= 768 ? 256 : 1024;
}
template <int DT> hipError_t backward_any(const NormBackward& p, hipStream_t s) {
    const uint32_t pieces = (uint32_t)ceil_div(p.cols, 8);
    auto on = [&](auto g, auto r) {
        constexpr int G = decltype(g)::value, R = decltype(r)::value;
        return launch(norm_backward_kernel<DT, G, R>, p.parts, G, p, s);
    };
    if (pieces <= 64) return on(Int<64>{}, Int<1>{});
    if (pieces <= 128) return on(Int<128>{}, Int<1>{});
    if (pieces <= 192) return on(Int<64>{}, Int<3>{});
    if (pieces <= 256) return on(Int<256>{}, Int<1>{});
    if (pieces <= 384) return on(Int<128>{}, Int<3>{});
    if (pieces <= 512) return on(Int<512>{}, Int<1>{});
    if (pieces <= 768) return on(Int<256>{}, Int<3>{});
    if (pieces <= 1024) return on(Int<1024>{}, Int<1>{});
    if (pieces <= 2048) return on(Int<1024>{}, Int<2>{});
    return on(Int<1024>{}, Int<0>{});
}

}  // namespace

uint32_t norm_backward_parts(uint32_t rows, uint32_t cols) {
    // as many work-groups as are resident at once, 2048 threads a CU, up to 1024, but two rows each
    // where there are 512 of those: every range is written, read and added once more
    const uint32_t resident = kComputeUnits * 2048u / backward_threads(cols);
    uint32_t parts = resident < 1024u ? resident : 1024u;
    const uint32_t two = (rows + 1) / 2 < 512u ? 512u : (rows + 1) / 2;
    if (parts > two) parts = two;
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
    return hipLaunchKernel(reinterpret_cast<const void*>(&column_sum_kernel), dim3((cols + 31) / 32), dim3(1024), args, 0, s);
}

}  // namespace q8
