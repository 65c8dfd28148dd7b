// Device helpers of the 8-bit operators: types, loads of eight values, sums over
// the threads of a row.
#pragma once

#include "q8_shim.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace q8 {

template <int V> struct Int { static constexpr int value = V; };

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
// the same at any address: the memory pipeline takes vector accesses at byte
// alignment, so rows may start anywhere
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
typedef f32x4 f32x4_at4 __attribute__((aligned(4)));
typedef uint32_t u32_at1 __attribute__((aligned(1)));
typedef u32x2 u32x2_at1 __attribute__((aligned(1)));
typedef u32x4 u32x4_at1 __attribute__((aligned(1)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));

// 16 bytes as they are loaded.  From any address: five dwords, those that hold the bytes, and the bytes
// once they have arrived, of which `at` of the first dword come before them.  No dword is read
// that holds none of the 16.
template <bool ODD> struct Raw {
    typedef u32x4 T;
    static __device__ __forceinline__ T load(const char* p) { return *reinterpret_cast<const u32x4_at1*>(p); }
    static __device__ __forceinline__ u32x4 value(const T& v, uint32_t) { return v; }
};
template <> struct Raw<true> {
    struct T { u32x4 w; uint32_t x; };
    static __device__ __forceinline__ T load(const char* p) {
        const char* first = (const char*)((uintptr_t)p & ~(uintptr_t)3);
        const char* last = (const char*)((uintptr_t)(p + 15) & ~(uintptr_t)3);
        return T{*reinterpret_cast<const u32x4_at4*>(first), *reinterpret_cast<const uint32_t*>(last)};
    }
    static __device__ __forceinline__ u32x4 value(const T& v, uint32_t at) {
        return u32x4{__builtin_amdgcn_alignbyte(v.w[1], v.w[0], at), __builtin_amdgcn_alignbyte(v.w[2], v.w[1], at),
                     __builtin_amdgcn_alignbyte(v.w[3], v.w[2], at), __builtin_amdgcn_alignbyte(v.x, v.w[3], at)};
    }
};

template <int DT> struct Type;
template <> struct Type<Q8_F32> {
    typedef float T;
    static __device__ __forceinline__ float get(const T* p) { return *p; }
    static __device__ __forceinline__ void put(T* p, float x) { *p = x; }
    static __device__ __forceinline__ float round(float x) { return x; }
    // eight values as they are in memory, and spread out
    struct Eight { f32x4 lo, hi; };
    static __device__ __forceinline__ Eight get8(const T* p) {
        return Eight{*reinterpret_cast<const f32x4_at4*>(p), *reinterpret_cast<const f32x4_at4*>(p + 4)};
    }
    static __device__ __forceinline__ void spread(const Eight& w, float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = w.lo[e]; v[4 + e] = w.hi[e]; }
    }
    static __device__ __forceinline__ void load8(const T* p, float (&v)[8]) { spread(get8(p), v); }
    static __device__ __forceinline__ Eight eight(const float (&v)[8]) {
        return Eight{f32x4{v[0], v[1], v[2], v[3]}, f32x4{v[4], v[5], v[6], v[7]}};
    }
    static __device__ __forceinline__ void put8(T* p, const Eight& w) {
        *reinterpret_cast<f32x4_at4*>(p) = w.lo;
        *reinterpret_cast<f32x4_at4*>(p + 4) = w.hi;
    }
    static __device__ __forceinline__ void store8(T* p, const float (&v)[8]) { put8(p, eight(v)); }
};
template <> struct Type<Q8_F16> {
    typedef _Float16 T;
    static __device__ __forceinline__ float get(const T* p) { return (float)*p; }
    static __device__ __forceinline__ void put(T* p, float x) { *p = (T)x; }
    static __device__ __forceinline__ float round(float x) { return (float)(T)x; }
    typedef u32x4 Eight;
    static __device__ __forceinline__ Eight get8(const T* p) { return *reinterpret_cast<const u32x4_at2*>(p); }
    static __device__ __forceinline__ void load8(const T* p, float (&v)[8]) { spread(get8(p), v); }
    static __device__ __forceinline__ void spread(const Eight& w, float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const f16x2 h = __builtin_bit_cast(f16x2, (uint32_t)w[e]);
            v[2 * e] = (float)h[0];
            v[2 * e + 1] = (float)h[1];
        }
    }
    static __device__ __forceinline__ uint32_t pair(float x, float y) {
        const f16x2 h = {(_Float16)x, (_Float16)y};
        return __builtin_bit_cast(uint32_t, h);
    }
    static __device__ __forceinline__ Eight eight(const float (&v)[8]) {
        return u32x4{pair(v[0], v[1]), pair(v[2], v[3]), pair(v[4], v[5]), pair(v[6], v[7])};
    }
    static __device__ __forceinline__ void put8(T* p, const Eight& w) { *reinterpret_cast<u32x4_at2*>(p) = w; }
    static __device__ __forceinline__ void store8(T* p, const float (&v)[8]) { put8(p, eight(v)); }
};
template <> struct Type<Q8_BF16> {
    typedef __bf16 T;
    static __device__ __forceinline__ float get(const T* p) { return (float)*p; }
    static __device__ __forceinline__ void put(T* p, float x) { *p = (T)x; }
    static __device__ __forceinline__ float round(float x) { return (float)(T)x; }
    typedef u32x4 Eight;
    static __device__ __forceinline__ Eight get8(const T* p) { return *reinterpret_cast<const u32x4_at2*>(p); }
    static __device__ __forceinline__ void load8(const T* p, float (&v)[8]) { spread(get8(p), v); }
    static __device__ __forceinline__ void spread(const Eight& w, float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = __builtin_bit_cast(float, (uint32_t)(w[e] << 16));
            v[2 * e + 1] = __builtin_bit_cast(float, (uint32_t)(w[e] & 0xffff0000u));
        }
    }
    static __device__ __forceinline__ uint32_t pair(float x, float y) {
        const f32x2 v = {x, y};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    }
    static __device__ __forceinline__ Eight eight(const float (&v)[8]) {
        return u32x4{pair(v[0], v[1]), pair(v[2], v[3]), pair(v[4], v[5]), pair(v[6], v[7])};
    }
    static __device__ __forceinline__ void put8(T* p, const Eight& w) { *reinterpret_cast<u32x4_at2*>(p) = w; }
    static __device__ __forceinline__ void store8(T* p, const float (&v)[8]) { put8(p, eight(v)); }
};

// Eight values of a row from column c; those past `cols` are 0 (c < cols).
template <int DT>
__device__ __forceinline__ void load_part(const typename Type<DT>::T* row, uint32_t c, uint32_t cols, float (&v)[8]) {
    if (cols - c >= 8) {
        Type<DT>::load8(row + c, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? Type<DT>::get(row + c + e) : 0.0f;
    }
}
template <int DT>
__device__ __forceinline__ void store_part(typename Type<DT>::T* row, uint32_t c, uint32_t cols, const float (&v)[8]) {
    if (cols - c >= 8) {
        Type<DT>::store8(row + c, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < cols) Type<DT>::put(row + c + e, v[e]);
    }
}

// v = v sx sw + add for integer sums v.  A sum has 31 bits, so a token's scale from 2^96 on could take it past FP32's
// range where the channel's brings it back: there the channel's comes first, and what passes the range then
// is a result that does.
template <int N>
__device__ __forceinline__ void finish(float (&v)[N], float sx, const float (&sw)[N], const float (&add)[N]) {
    const bool last = sx >= 0x1p96f;
    if (__builtin_expect(__any(last), 0)) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = __builtin_fmaf(v[e] * (last ? sw[e] : sx), last ? sx : sw[e], add[e]);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = __builtin_fmaf(v[e] * sx, sw[e], add[e]);
    }
}

// |x| as an integer that orders like it, infinities and then NaN last.
__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}

// Sum of f and maximum of u over a wave, in every lane, in a fixed order.
__device__ __forceinline__ void wave_sum_max(float& f, uint32_t& u) {
    auto step = [&](uint32_t fo, uint32_t uo) __attribute__((always_inline)) {
        f += __builtin_bit_cast(float, fo);
        u = u > uo ? u : uo;
    };
    auto bits = [&]() __attribute__((always_inline)) { return __builtin_bit_cast(uint32_t, f); };
    step(dpp<0xb1>(bits()), dpp<0xb1>(u));     // lane ^ 1
    step(dpp<0x4e>(bits()), dpp<0x4e>(u));     // lane ^ 2
    step(dpp<0x141>(bits()), dpp<0x141>(u));   // the other four of eight
    step(dpp<0x140>(bits()), dpp<0x140>(u));   // the other eight of sixteen
    step((uint32_t)__shfl_xor((int)bits(), 16), (uint32_t)__shfl_xor((int)u, 16));
    step((uint32_t)__shfl_xor((int)bits(), 32), (uint32_t)__shfl_xor((int)u, 32));
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
__device__ __forceinline__ u32x2 bytes8(const float (&u)[8], const Scale& s) {
    uint32_t q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = to8(u[e], s);
    return u32x2{q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24, q[4] | q[5] << 8 | q[6] << 16 | q[7] << 24};
}

template <bool HALF> __device__ __forceinline__ uint32_t pair16(float x, float y) {
    return HALF ? Type<Q8_F16>::pair(x, y) : Type<Q8_BF16>::pair(x, y);
}

// x = hi + mid + lo in BF16, each cut off where the next one goes on: both differences are exact,
// and three terms of 8 bits hold the 24 of FP32, of all x from 2^-110 on (below, the last term's bits pass BF16's
// smallest step, 2^-133).  Infinities and NaN stay in the first term.
// The terms are the upper halves of b.
__device__ __forceinline__ void three(float x, uint32_t (&b)[3]) {
    x = __builtin_canonicalizef(x);     // a NaN has a bit in the first term
    b[0] = __builtin_bit_cast(uint32_t, x);
    const float r = magnitude(x) < 0x7f800000u ? x - __builtin_bit_cast(float, b[0] & 0xffff0000u) : 0.0f;
    b[1] = __builtin_bit_cast(uint32_t, r);
    b[2] = __builtin_bit_cast(uint32_t, r - __builtin_bit_cast(float, b[1] & 0xffff0000u));
}
// The upper halves of two.
__device__ __forceinline__ uint32_t uppers(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }

// Half precision keeps 2^-14 .. 2^15 with all its bits, and the weights' values are
// q scale: a power of two brings the largest scale to 2^7 .. 2^8 (127 times it still fits),
// and the product is multiplied by its inverse in 32 bits.  The largest finite scale over a
// work-group:
template <int THREADS> __device__ __forceinline__ uint32_t largest(const float* scale, uint32_t count, uint32_t (&red)[THREADS / 64]) {
    uint32_t top = 0;
    for (uint32_t i = threadIdx.x; i < count; i += THREADS * 4) {
        uint32_t a[4];      // four loads at once; the last one again past the end
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] = magnitude(scale[min(i + k * THREADS, count - 1)]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (a[k] < 0x7f800000u) top = top > a[k] ? top : a[k];
    }
    float none = 0.0f;
    wave_sum_max(none, top);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) top = top > red[w] ? top : red[w];
    return top;
}
// 2^-e and 2^e
__device__ __forceinline__ void powers(uint32_t top, float& down, float& up) {
    int e = (int)(top >> 23) - 127 - 7;           // scale in [2^(e + 7), 2^(e + 8))
    e = e < -126 ? -126 : e > 126 ? 126 : e;      // both powers stay normal
    down = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
    up = __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
}

constexpr int XCDS = 8;
// Workgroups go round the XCDs one by one: consecutive tiles to one XCD instead, so that
// its L2 serves their shared rows.
__device__ __forceinline__ uint32_t xcd_order(uint32_t id, uint32_t total) {
    const uint32_t x = id % XCDS, q = total / XCDS, r = total % XCDS;
    return x * q + (x < r ? x : r) + id / XCDS;
}

}  // namespace q8
