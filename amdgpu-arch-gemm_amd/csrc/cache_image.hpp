// What the kernels for many new tokens share (gfx950): images of 64 keys and values, and the joining of pieces.
#pragma once

#include "cache_attention_device.hpp"

namespace q8 {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// 64 keys and values of one sequence and head as 16-bit values, with the keys' scales: what a step multiplies.
// Keys lie in an image by rows of a key's values, values by rows of one value's keys, each row 16 bytes longer than what it
// holds: reads of 16 bytes down a column go by 16 lanes a cycle (0-3, 12-15, 20-27 and so on), whose rows then meet all 64 banks, and
// every place of a lane's is its first one plus a constant.  The eight keys of a piece
// of the values are those that a lane has of each 16 after the scores (0-3, 8-11 and 4-7, 12-15).
template <int DT, int DP> struct Image {
    static constexpr bool QH = DT == Q8_F16, VH = DT != Q8_F32;       // half precision, not BF16
    static constexpr int KEY_ROW = DP * 2 + 16, VALUE_ROW = 128 + 16, KEYS = 64 * KEY_ROW, VALUES = DP * VALUE_ROW;
    // after them 64 scales of keys, with the scores' factor, 64 of values, and a bit for each key that is there
    static constexpr int SCALES = KEYS + VALUES, BYTES = SCALES + 1024;
    static_assert(BYTES == (int)image_bytes(DP), "the workspace's images");
    // Where a lane reads: key lane % 32 of the first 32, values lane % 32.
    static __device__ __forceinline__ uint32_t key_at(int n, int half) { return n * KEY_ROW + half * 16; }
    static __device__ __forceinline__ uint32_t value_at(int n, int half) { return KEYS + n * VALUE_ROW + half * 16; }
};

// The units of an image that one of THREADS threads makes, keys' or values', from memory by way of registers.
template <int DT, int DP, int THREADS> struct Units {
    typedef Image<DT, DP> F;
    static constexpr int KEY_UNITS = 64 * (DP / 16), KEY_LOADS = (KEY_UNITS + THREADS - 1) / THREADS;       // 16 bytes each
    static constexpr int VALUE_UNITS = 8 * (DP / 4), VALUE_LOADS = (VALUE_UNITS + THREADS - 1) / THREADS;   // eight keys of four values
    static constexpr int KEY_STEP = THREADS / (DP / 16), PART_STEP = THREADS / (DP / 4);
    static constexpr int HELD = KEY_LOADS * 4 > VALUE_LOADS * 8 ? KEY_LOADS * 4 : VALUE_LOADS * 8;
    static __device__ __forceinline__ uint32_t key_at(int i) { return i / (DP / 16) * F::KEY_ROW + i % (DP / 16) * 32; }
    static __device__ __forceinline__ uint32_t value_at(int i) { return F::KEYS + i % (DP / 4) * 4 * F::VALUE_ROW + i / (DP / 4) * 16; }
    // offset: of the keys' rows
    static __device__ __forceinline__ void load_keys(const Paged& c, const uint64_t* offset, int i, uint32_t* held) {
#pragma unroll
        for (int x = 0; x < KEY_LOADS; ++x) {
            const int u = i + x * THREADS, key = u / (DP / 16) % 64, d = u % (DP / 16) * 16;
            const u32x4 w = *reinterpret_cast<const u32x4*>(c.k + offset[key] + (d < (int)c.pitch ? d : 0));
#pragma unroll
            for (int e = 0; e < 4; ++e) held[4 * x + e] = w[e];
        }
    }
    static __device__ __forceinline__ void load_values(const Paged& c, const uint64_t* offset, int i, uint32_t* held) {
#pragma unroll
        for (int x = 0; x < VALUE_LOADS; ++x) {
            const int u = i + x * THREADS, part = u / (DP / 4) % 8, d = u % (DP / 4) * 4, first = part / 2 * 16 + part % 2 * 4;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                held[8 * x + e] = *reinterpret_cast<const uint32_t*>(c.v + offset[first + (e >> 2) * 8 + (e & 3)] + (d < (int)c.pitch ? d : 0));
        }
    }
    // `at`: key_at(i) or value_at(i) in the image at `to`
    static __device__ __forceinline__ void store_keys(char* to, uint32_t at, int i, const uint32_t* held) {
#pragma unroll
        for (int x = 0; x < KEY_LOADS; ++x) {
            if (KEY_UNITS % THREADS && i + x * THREADS >= KEY_UNITS) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u32x2 w0 = four<F::QH>(kept(held[4 * x + 2 * h])), w1 = four<F::QH>(kept(held[4 * x + 2 * h + 1]));
                *reinterpret_cast<u32x4*>(to + at + x * KEY_STEP * F::KEY_ROW + h * 16) = u32x4{w0[0], w0[1], w1[0], w1[1]};
            }
        }
    }
    static __device__ __forceinline__ void store_values(char* to, uint32_t at, int i, const uint32_t* held) {
#pragma unroll
        for (int x = 0; x < VALUE_LOADS; ++x) {
            if (VALUE_UNITS % THREADS && i + x * THREADS >= VALUE_UNITS) break;
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = kept(held[8 * x + e]);
            u32x4 r[4];
            columns<F::VH>(w, r);
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<u32x4*>(to + at + x * PART_STEP * 16 + j * F::VALUE_ROW) = r[j];
        }
    }
};

// This lane's key of the 64 from k: its row (another key's where it is not there, if one is), and a bit for each that is there.
__device__ __forceinline__ uint64_t find_row(const Paged& c, uint32_t kv, int k, int end, int page, int64_t& row) {
    const uint32_t lane = threadIdx.x & 63, key = (uint32_t)k + lane;
    page = (int)key < end && (uint32_t)kept((uint32_t)page) < c.pages ? page : -1;
    const uint64_t there = __ballot(page >= 0);
    if (!there) return 0;
    row = ((int64_t)page * c.heads + kv) * c.page_tokens + (key - divide(key, c.page) * c.page_tokens);
    const int some = __builtin_ctzll(there);
    const int64_t other = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(row >> 32), some) << 32 |
                                    (uint32_t)__builtin_amdgcn_readlane((int)row, some));
    row = page < 0 ? other : row;
    return there;
}

// The tile of ROWS rows of a work-group; its keys begin at an image's.
template <int ROWS> __device__ __forceinline__ bool find_rows(const AttentionArgs& g, Place& t) {
    // the last tiles of a sequence see the most keys and come first
    if (!find_tile(g, g.slots - 1 - blockIdx.x / g.a.at.heads, ROWS, t)) return false;
    t.begin &= ~63;
    return true;
}

// A row's result, or its sums of one of several pieces: a lane has of each 32 values 8 i + 4 half .. + 3, i = 0 .. 3.
template <int DT, int DP>
__device__ __forceinline__ void put_row(const AttentionArgs& g, const Row& at, uint32_t piece, int pieces, int half, const Reference& r, float l,
                                        const f32x16 (&o)[DP / 32]) {
    typedef typename Type<DT>::T T;
    const Attention& a = g.a;
    const uint64_t to = at.row * a.heads + at.head;
    if (pieces > 1) {       // join_kernel's
        const uint64_t own = (uint64_t)piece * a.at.tokens * a.heads + to;
        float R;
        const float up = without_rest(r, R, l), down = settle(R, l) * up;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<f32x4*>(g.sums + own * DP + d * 32 + i * 2 + half * 4) =
                    f32x4{o[d][i] * down, o[d][i + 1] * down, o[d][i + 2] * down, o[d][i + 3] * down};
        if (half == 0) {
            g.stats[2 * own] = R;
            g.stats[2 * own + 1] = l;
        }
        return;
    }
    const float part = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = (T*)a.out + at.row * a.ldo + at.head * a.at.dim;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t x = d * 32 + (i >> 2) * 8 + half * 4 + (i & 3);
            if (x < a.at.dim) Type<DT>::put(out + x, o[d][i] * part);
        }
    if (a.lse && half == 0) a.lse[to] = l == 0.0f ? -__builtin_huge_valf() : (r.far.base + (r.far.rest + __builtin_log2f(l))) * kLn2;
}

// The pieces' sums of a tile's rows: DP / 8 threads a row, 2048 / DP rows a work-group.  (A work-group of the kernel before
// that finishes a tile and adds them alone reads for longer than all work-groups together: 64 tokens over 8192 keys,
// 32 pieces, 195 us.)
template <int DT, int DP, int ROWS> __global__ void __launch_bounds__(256) join_kernel(const AttentionArgs g) {
    typedef typename Type<DT>::T T;
    constexpr int ACROSS = DP / 8;
    const Attention& a = g.a;
    const Paged& c = a.at;
    const uint32_t kv = blockIdx.x % c.heads;
    Place t;
    if (!find_rows<ROWS>(g, t)) return;
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

template <typename K> hipError_t launch(K kernel, dim3 groups, uint32_t threads, const AttentionArgs& g, hipStream_t s) {
    void* args[] = {const_cast<AttentionArgs*>(&g)};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), groups, dim3(threads), args, 0, s);
}

}  // namespace q8
