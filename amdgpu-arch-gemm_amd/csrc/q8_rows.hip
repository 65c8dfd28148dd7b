// Row kernels of the 8-bit operators (gfx950): quantisation, the root-mean-square
// norm with the residual's addition and its 8-bit result, that norm's gradients,
// and the restoring of 8-bit rows.  All are one pass over their data and bounded
// by memory.
//
// A row belongs to G threads, eight values each at a time, and stays in
// registers between its sums and its stores.  Rows may start at any address (see
// q8_device.hpp).  A row's last piece starts where the row has eight values left: those that the
// piece before it has too count once in sums and are stored twice, the same, so that no access is
// shorter than eight values (1000 x 999, F16: 6.3 -> 3.9 us).  Rows of fewer than eight values, or
// of more than the registers hold, have kernels that go by elements at the end and read twice.
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
// Piece i of a row for one of its G threads.
struct Piece {
    uint32_t c, twice;   // first column; so many of its values are the piece before's
    bool on;
};
template <int G> __device__ __forceinline__ Piece piece_of(int i, uint32_t lane, uint32_t cols) {
    const uint32_t c = (uint32_t)(i * G + (int)lane) * 8;
    Piece p;
    p.on = c < cols;
    p.c = min(c, cols - 8);
    p.twice = c - p.c;
    return p;
}
__device__ __forceinline__ u32x2 bytes8(const float (&u)[8], const Scale& s) {
    uint32_t q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = to8(u[e], s);
    return u32x2{q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24, q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24};
}

// Quantisation (NORM == false) and the norm, R pieces a thread.  hidden leaves after the sums: it
// may be x or the residual, whose last values two threads read.
template <int DT, bool NORM, int G, int R>
__global__ void __launch_bounds__(G < 256 ? 256 : G) quantize_kernel(const Quantize p) {
    constexpr int WG = G < 256 ? 256 : G, ROWS = WG / G;
    typedef Type<DT> Y;
    typedef typename Y::T T;
    __shared__ float redf[2][WG / 64];
    __shared__ uint32_t redu[2][WG / 64];
    const uint32_t lane = threadIdx.x % G;
    const T* gain = (const T*)p.gain;
    int set = 0;
    for (uint64_t r0 = (uint64_t)blockIdx.x * ROWS; r0 < p.rows; r0 += (uint64_t)gridDim.x * ROWS, set ^= 1) {
        const uint64_t row = r0 + threadIdx.x / G;
        const bool on = row < p.rows;
        const T* x = (const T*)p.x + row * p.ldx;
        const T* res = NORM && p.residual ? (const T*)p.residual + row * p.ldr : nullptr;
        T* hid = NORM && p.hidden ? (T*)p.hidden + row * p.ldh : nullptr;
        float v[R][8];
        typename Y::Eight hold[NORM ? R : 1];
        float sum = 0.0f;
        uint32_t top = 0;
        // all loads of the row before its first sum
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const Piece c = piece_of<G>(i, lane, p.cols);
            if (!on || !c.on) continue;
            Y::load8(x + c.c, v[i]);
            if (NORM && res) {
                float w[8];
                Y::load8(res + c.c, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] = Y::round(v[i][e] + w[e]);
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const Piece c = piece_of<G>(i, lane, p.cols);
            if (!on || !c.on) continue;
            if constexpr (NORM) {
                hold[i] = Y::eight(v[i]);
                float g[8];
                Y::load8(gain + c.c, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float h = (uint32_t)e < c.twice ? 0.0f : v[i][e];
                    sum = __builtin_fmaf(h, h, sum);
                    v[i][e] *= g[e];    // u
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t a = magnitude(v[i][e]);
                top = top > a ? top : a;
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
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const Piece c = piece_of<G>(i, lane, p.cols);
            if (!on || !c.on) continue;
            if (NORM && hid) Y::put8(hid + c.c, hold[i]);
            *reinterpret_cast<u32x2_at1*>(q + c.c) = bytes8(v[i], s);
        }
    }
}

// The same for rows of fewer than eight values and for rows longer than registers hold: each piece is
// read a second time after the sums.
template <int DT, bool NORM, int G>
__global__ void __launch_bounds__(G < 256 ? 256 : G) quantize_any_kernel(const Quantize p) {
    constexpr int WG = G < 256 ? 256 : G, ROWS = WG / G;
    typedef typename Type<DT>::T T;
    __shared__ float redf[2][WG / 64];
    __shared__ uint32_t redu[2][WG / 64];
    const uint32_t lane = threadIdx.x % G;
    const T* gain = (const T*)p.gain;
    int set = 0;
    for (uint64_t r0 = (uint64_t)blockIdx.x * ROWS; r0 < p.rows; r0 += (uint64_t)gridDim.x * ROWS, set ^= 1) {
        const uint64_t row = r0 + threadIdx.x / G;
        const bool on = row < p.rows;
        const T* x = (const T*)p.x + row * p.ldx;
        const T* res = NORM && p.residual ? (const T*)p.residual + row * p.ldr : nullptr;
        T* hid = NORM && p.hidden ? (T*)p.hidden + row * p.ldh : nullptr;
        float sum = 0.0f;
        uint32_t top = 0;
        auto first = [&](uint32_t c, float (&v)[8]) __attribute__((always_inline)) {
            load_part<DT>(x, c, p.cols, v);
            if (NORM && res) {
                float w[8];
                load_part<DT>(res, c, p.cols, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = Type<DT>::round(v[e] + w[e]);
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
        for (uint32_t c = lane * 8; on && c < p.cols; c = next_column(c, G * 8, p.cols)) {
            float v[8];
            first(c, v);
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
        for (uint32_t c = lane * 8; on && c < p.cols; c = next_column(c, G * 8, p.cols)) {
            float v[8];
            if (hid) load_part<DT>(hid, c, p.cols, v);   // x may be gone: hidden may be x itself
            else first(c, v);
            weigh(c, v);
            const u32x2 b = bytes8(v, s);
            if (p.cols - c >= 8) {
                *reinterpret_cast<u32x2_at1*>(q + c) = b;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < p.cols) q[c + e] = (int8_t)(b[e / 4] >> (8 * (e % 4)));
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
        if (p.cols < 8) {
            if (lane < p.cols) Type<DT>::put(y + lane, (float)q[lane] * s);
            continue;
        }
        for (uint32_t n = lane * 8; n < p.cols; n = next_column(n, G * 8, p.cols)) {
            const uint32_t c = min(n, p.cols - 8);
            float v[8];
            const u32x2 w = *reinterpret_cast<const u32x2_at1*>(q + c);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)(w[e / 4] >> (8 * (e % 4))) * s;
            Type<DT>::store8(y + c, v);
        }
    }
}

// dx and, for the work-group's rows blockIdx.x, blockIdx.x + parts, ..., the
// sums of dn xhat for each column: a thread has the same columns in every row, so
// they stay in its registers and are added in row order.  dx leaves after the sums and dres is read before
// them: dx may be dn or dres.
template <int DT, int G, int R>
__global__ void __launch_bounds__(G) norm_backward_kernel(const NormBackward p) {
    typedef Type<DT> Y;
    typedef typename Y::T T;
    __shared__ float redf[2][G / 64];
    __shared__ uint32_t redu[2][G / 64];
    const uint32_t lane = threadIdx.x;
    const T* gain = (const T*)p.gain;
    float acc[R][8];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[i][e] = 0.0f;
    const float per = 1.0f / (float)p.cols;
    int set = 0;
    for (uint64_t row = blockIdx.x; row < p.rows; row += p.parts, set ^= 1) {
        const T* dn = (const T*)p.dn + row * p.lddn;
        const T* hid = (const T*)p.hidden + row * p.ldh;
        const T* res = p.dres ? (const T*)p.dres + row * p.lddr : nullptr;
        T* dx = (T*)p.dx + row * p.lddx;
        const float rstd = p.rstd[row];
        float u[R][8], xh[R][8];
        typename Y::Eight d[R];
        float sum = 0.0f;
        uint32_t none = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const Piece c = piece_of<G>(i, lane, p.cols);
            if (!c.on) continue;
            float g[8];
            Y::load8(dn + c.c, u[i]);
            Y::load8(hid + c.c, xh[i]);
            if (res) d[i] = Y::get8(res + c.c);
            Y::load8(gain + c.c, g);
            // u = dn gain, xhat; and dn xhat for the gain's gradient
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                xh[i][e] *= rstd;
                acc[i][e] = __builtin_fmaf(u[i][e], xh[i][e], acc[i][e]);
                u[i][e] *= g[e];
                sum = __builtin_fmaf((uint32_t)e < c.twice ? 0.0f : u[i][e], (uint32_t)e < c.twice ? 0.0f : xh[i][e], sum);
            }
        }
        row_sum_max<G, G>(sum, none, redf, redu, set);
        const float mean = sum * per;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const Piece c = piece_of<G>(i, lane, p.cols);
            if (!c.on) continue;
            float y[8];
            if (res) Y::spread(d[i], y);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float z = rstd * (u[i][e] - xh[i][e] * mean);
                y[e] = res ? z + y[e] : z;
            }
            Y::store8(dx + c.c, y);
        }
    }
    if (p.dgain) {
        float* part = p.partial + (uint64_t)blockIdx.x * p.cols;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const Piece c = piece_of<G>(i, lane, p.cols);
            if (c.on) Type<Q8_F32>::store8(part + c.c, acc[i]);
        }
    }
}

// The same for rows of fewer than eight values and for rows longer than registers hold.
template <int DT, int G> __global__ void __launch_bounds__(G) norm_backward_any_kernel(const NormBackward p) {
    typedef typename Type<DT>::T T;
    __shared__ float redf[2][G / 64];
    __shared__ uint32_t redu[2][G / 64];
    const uint32_t lane = threadIdx.x;
    const T* gain = (const T*)p.gain;
    const float per = 1.0f / (float)p.cols;
    float* part = p.dgain ? p.partial + (uint64_t)blockIdx.x * p.cols : nullptr;
    int set = 0;
    for (uint64_t row = blockIdx.x; row < p.rows; row += p.parts, set ^= 1) {
        const T* dn = (const T*)p.dn + row * p.lddn;
        const T* hid = (const T*)p.hidden + row * p.ldh;
        const T* res = p.dres ? (const T*)p.dres + row * p.lddr : nullptr;
        T* dx = (T*)p.dx + row * p.lddx;
        const float rstd = p.rstd[row];
        float sum = 0.0f;
        uint32_t none = 0;
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
            }
        };
        // the column sums stay in the partial row, each entry its own thread's
        for (uint32_t c = lane * 8; c < p.cols; c = next_column(c, G * 8, p.cols)) {
            float u[8], xh[8], a[8] = {};
            if (part && row != blockIdx.x) load_part<Q8_F32>(part, c, p.cols, a);
            first(c, u, xh, a);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(u[e], xh[e], sum);
            if (part) store_part<Q8_F32>(part, c, p.cols, a);
        }
        row_sum_max<G, G>(sum, none, redf, redu, set);
        for (uint32_t c = lane * 8; c < p.cols; c = next_column(c, G * 8, p.cols)) {
            float u[8], xh[8], a[8] = {}, d[8] = {};
            first(c, u, xh, a);
            if (res) load_part<DT>(res, c, p.cols, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float z = rstd * (u[e] - xh[e] * (sum * per));
                d[e] = res ? z + d[e] : z;
            }
            store_part<DT>(dx, c, p.cols, d);
        }
    }
}

// dgain_j = the parts' sums in part order: 32 columns a work-group, 32 slices of parts that meet in
// LDS, so that few columns still reach many CUs (512 x 999: 64 columns and 16 slices 6.8 us).  The grid has two
// dimensions, as one ends at 2^32 work-items, 2^27 columns.  (A loop over a work-group's columns costs more: its
// loads wait for one another then, 1000 x 999 with it 12.2 us for 8.7.)
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* partial, float* dgain, uint32_t parts, uint32_t cols) {
    __shared__ float red[32][33];
    const uint32_t lane = threadIdx.x % 32, slice = threadIdx.x / 32, c = (blockIdx.y * kMostGroups + blockIdx.x) * 32 + lane;
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

// The threads of a row and their pieces of eight values: the least G * R that holds the row, with the
// most threads up to 512.  (F16, G x R: 16384 x 8192 512 x 2 178 us, 5.3 TB/s, 1024 x 1 202, 256 x 4 206.
// 1000 x 4097: 256 x 3 8.5 us, 512 x 2 9.4, 1024 x 1 11.9.  8192 x 6001: 256 x 3 81 us, 512 x 2 85.  1 x 4096:
// 512 x 1 2.9 us, 128 x 4 4.5.)
template <int DT, bool NORM> hipError_t quantize_any(const Quantize& p, hipStream_t s) {
    const uint32_t pieces = (uint32_t)ceil_div(p.cols, 8);
    auto on = [&](auto g, auto r) {
        constexpr int G = decltype(g)::value, R = decltype(r)::value;
        return launch(quantize_kernel<DT, NORM, G, R>, groups_for(p.rows, G < 256 ? 256 / G : 1), G < 256 ? 256 : G, p, s);
    };
    if (p.cols < 8) return launch(quantize_any_kernel<DT, NORM, 64>, groups_for(p.rows, 4), 256, p, s);
    if (pieces <= 64) return on(Int<64>{}, Int<1>{});
    if (pieces <= 128) return on(Int<128>{}, Int<1>{});
    if (pieces <= 192) return on(Int<64>{}, Int<3>{});
    if (pieces <= 256) return on(Int<256>{}, Int<1>{});
    if (pieces <= 384) return on(Int<128>{}, Int<3>{});
    if (pieces <= 512) return on(Int<512>{}, Int<1>{});
    if (pieces <= 768) return on(Int<256>{}, Int<3>{});
    if (pieces <= 1024) return on(Int<512>{}, Int<2>{});
    if (pieces <= 1536) return on(Int<512>{}, Int<3>{});
    if (pieces <= 2048) return on(Int<512>{}, Int<4>{});
    if (pieces <= 4096) return on(Int<1024>{}, Int<4>{});
    return launch(quantize_any_kernel<DT, NORM, 1024>, groups_for(p.rows, 1), 1024, p, s);
}

template <int DT> hipError_t dequantize_any(const Dequantize& p, hipStream_t s) {
    if (p.cols <= 512) return launch(dequantize_kernel<DT, 64>, groups_for(p.rows, 4), 256, p, s);
    return launch(dequantize_kernel<DT, 256>, groups_for(p.rows, 1), 256, p, s);
}

// Row ranges that a column's sum is taken over first, one work-group each: two a CU that has 512
// threads (BF16, 16384 x 4096: 256 / 512 / 1024 ranges 118 / 98 / 116 us, 5.5 TB/s; 16384 x 8192 207 / 194 / 205;
// 1000 x 999 10.3 / 8.0 / 10.8): each range is written, read and added once more.  Threads whose last pieces are empty
// cost little, so there are no kernels for the widths between (2^27 BF16 values in rows of 4096 5.5 TB/s, 5120 5.3, 6144 5.6,
// 8192 5.6, 10240 5.2, 12288 5.2, 16384 5.2).
constexpr uint32_t kMostParts = 512;
template <int DT> hipError_t backward_any(const NormBackward& p, hipStream_t s) {
    const uint32_t pieces = (uint32_t)ceil_div(p.cols, 8);
    auto on = [&](auto g, auto r) {
        constexpr int G = decltype(g)::value, R = decltype(r)::value;
        return launch(norm_backward_kernel<DT, G, R>, p.parts, G, p, s);
    };
    if (p.cols < 8) return launch(norm_backward_any_kernel<DT, 64>, p.parts, 64, p, s);
    if (pieces <= 64) return on(Int<64>{}, Int<1>{});
    if (pieces <= 128) return on(Int<128>{}, Int<1>{});
    if (pieces <= 256) return on(Int<256>{}, Int<1>{});
    if (pieces <= 512) return on(Int<512>{}, Int<1>{});
    if (pieces <= 1024) return on(Int<512>{}, Int<2>{});
    if (pieces <= 2048) return on(Int<1024>{}, Int<2>{});
    return launch(norm_backward_any_kernel<DT, 1024>, p.parts, 1024, p, s);
}

}  // namespace

uint32_t norm_backward_parts(uint32_t rows) { return rows < kMostParts ? rows : kMostParts; }

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
    // at most kMostGroups x 2^7 work-groups, and kMostGroups of them wherever y is not 1: no column index passes 32 bits
    const uint32_t x = groups_for(cols, 32), y = (uint32_t)ceil_div(ceil_div(cols, 32), x);
    return hipLaunchKernel(reinterpret_cast<const void*>(&column_sum_kernel), dim3(x, y), dim3(1024), args, 0, s);
}

hipError_t prepare_rows() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(&column_sum_kernel));
}

}  // namespace q8
