// Attention of prompts and long chunks over the paged cache (gfx950), in 16-bit types, heads of up to 128 values.
#include "cache_image.hpp"

namespace q8 {
namespace {

constexpr int BUFFER_RSRC_WORD3 = 0x00020000;
constexpr int kWaves = 4, kThreads = 64 * kWaves, kRows = 64 * kWaves, kImages = 4;

// 64 keys from a multiple of 64, of one sequence and one of the cache's heads, as an image: 2.3 bytes written for each read, bounded
// by that (4 sequences of up to 8192 keys, 8 heads of 128: 33 us, 4.4 TB/s).  Each is read again by every 256 rows of the sequence.
template <int DT, int DP> __global__ void __launch_bounds__(256) image_kernel(const AttentionArgs g) {
    typedef Image<DT, DP> F;
    typedef Units<DT, DP, 128> U;
    __shared__ uint64_t offset[4][64];
    const Attention& a = g.a;
    const Paged& c = a.at;
    const uint32_t step = blockIdx.x % g.images_each, of = blockIdx.x / g.images_each, kv = of % c.heads, b = of / c.heads;
    const int tokens = max(chunk_end(c, b) - chunk_begin(c, b), 0), length = max(c.lengths[b], 0), k = (int)step * 64;
    const uint32_t rows = (uint32_t)tokens * a.group;
    const int end = (int)min((uint32_t)length, c.width * c.page_tokens);
    // the first key that the chunk's first token sees
    const int begin = a.window ? (int)max((int64_t)0, (int64_t)length - tokens - a.window + 1) : 0;
    if (rows <= g.least || rows > g.most || k >= end || k + 64 <= begin) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    char* image = g.images + (uint64_t)blockIdx.x * F::BYTES;
    int64_t row = 0;
    const int page = c.table[(uint64_t)b * c.table_ld + divide((uint32_t)min(k + lane, end - 1), c.page)];
    const uint64_t there = find_row(c, kv, k, end, page, row);
    if (wave == 0 && lane == 0) *reinterpret_cast<uint64_t*>(image + F::SCALES + 512) = there;
    // of keys none of which is there zeros, as what the workspace holds may be no numbers
    offset[wave][lane] = (uint64_t)row * c.pitch;
    __builtin_amdgcn_wave_barrier();
    if (wave == 0) *reinterpret_cast<float*>(image + F::SCALES + lane * 4) = there ? c.k_scale[row] * (a.scale * kLog2e) : 0.0f;
    if (wave == 2) *reinterpret_cast<float*>(image + F::SCALES + 256 + lane * 4) = there ? c.v_scale[row] : 0.0f;
    uint32_t held[U::HELD] = {};
    if (wave < 2) {
        if (there) U::load_values(c, offset[wave], tid, held);
        U::store_values(image, U::value_at(tid), tid, held);
    } else {
        if (there) U::load_keys(c, offset[wave], tid - 128, held);
        U::store_keys(image, U::key_at(tid - 128), tid - 128, held);
    }
}

// 1024 bytes, 16 a lane, to LDS.  The assembly form, since the compiler would wait for it before every read of LDS; the
// step's barrier waits.
__device__ __forceinline__ void to_lds(__amdgpu_buffer_rsrc_t rsrc, uint32_t lds, uint32_t lane_at, uint32_t at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" :: "s"(lds), "v"(lane_at), "s"(rsrc), "s"(at) : "memory");
}

// d = a b + d on the matrix cores.  In assembly, which alone says what lies in the accumulation half of the register file: the
// results of the second product and the queries, 192 registers of a wave, since it has 64 rows.  The compiler does not know how
// long a result takes (11 wait states): `settled` is between a product and what reads it.  A turn's scores come before its results,
// so that they are long done when the turn ends.
template <bool H> __device__ __forceinline__ void scores(u32x4 key, u32x4 query, f32x16& d, bool first) {
    if (first) {
        if constexpr (H) asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(d) : "v"(key), "a"(query));
        else asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(d) : "v"(key), "a"(query));
    } else {
        if constexpr (H) asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(d) : "v"(key), "a"(query));
        else asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(key), "a"(query));
    }
}
__device__ __forceinline__ void results(u32x4 value, u32x4 weight, f32x16& d) {
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(d) : "v"(value), "v"(weight));
}
__device__ __forceinline__ void settled(f32x16& d) { asm volatile("s_nop 15" : "+v"(d)); }
__device__ __forceinline__ void settled_acc(f32x16& d) { asm volatile("s_nop 15\n\ts_nop 15" : "+a"(d)); }

// Two values in half precision.  In assembly, as the compiler would round the products that they are by mixed instructions, which
// take twice as long.
__device__ __forceinline__ uint32_t halved(float x, float y) {
    uint32_t r;
    asm("v_cvt_pk_f16_f32 %0, %1, %2" : "=v"(r) : "v"(x), "v"(y));
    return r;
}
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
// Of two pairs of weights the larger ones, as integers: negative ones are larger yet.
__device__ __forceinline__ uint32_t larger(uint32_t x, uint32_t y) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, x), __builtin_bit_cast(u16x2, y)));
}
// Whether one of the largest is 2^15 or more, negative or no number.
__device__ __forceinline__ bool too_large(uint32_t m) { return ((m + 0x08000800u | m) & 0x80008000u) != 0; }

// A wave has 64 rows, A and B of 32, so that keys and values are read from LDS once for both.  (8192 tokens of 32 heads of 128, BF16:
// 633 us, 0.87 PFLOP/s, with the images' 14; eight waves of 32 rows on the same images 680; many_kernel 719; a large library product
// 1.2 PFLOP/s.  A turn of 16 matrix and some 100 vector instructions takes about 1200 cycles, without bank conflicts.  Matrix instructions
// are busy 41% of the cycles and vector instructions 43%: the two hardly overlap.  A wave is alone on its SIMD, for its registers, and a turn's
// scores are one chain of products through one accumulator; which of the two keeps the units apart was not measured.)  For each 32 keys h there are two turns of 16 matrix instructions (heads of 128), between each two of which
// are the vector instructions of one or two weights of the other rows:
//     scores of B(h), results of B(h - 1)   with the weights of A(h)
//     scores of A(h + 1), results of A(h)   with the weights of B(h)
// Keys and values of the next 32 are read in the first turn as the registers of these become free.
template <int DT, int DP> __global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const AttentionArgs g) {
    typedef Image<DT, DP> F;
    typedef typename Type<DT>::T T;
    constexpr int S = DP / 16, D = DP / 32, PRODUCTS = S + 2 * D;
    __shared__ __attribute__((aligned(1024))) char lds[kImages * F::BYTES];
    __shared__ Far fars[kWaves][2][32];
    const Attention& a = g.a;
    const Paged& c = a.at;
    const uint32_t kv = blockIdx.x % c.heads, piece = blockIdx.y;
    Place t;
    if (!find_rows<kRows>(g, t)) return;
    const int pieces = max(1, pieces_of(t, g.piece));
    if ((int)piece >= pieces) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, half = lane >> 5;
    const int begin = t.begin + (int)(piece * g.piece), end = piece_end(t, begin, g.piece);

    // Images on their way: a quarter of each by this wave.  begin + 64 * (image's number) is its first key.
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    char* first_image = g.images + ((uint64_t)t.b * c.heads + kv) * g.images_each * F::BYTES;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(first_image, (short)0, (int)(g.images_each * F::BYTES), BUFFER_RSRC_WORD3);
    constexpr int LOADS = F::BYTES / 1024, EACH = LOADS / kWaves, REST = LOADS % kWaves;      // wave 0 has the rest too
    auto load = [&](int k) __attribute__((always_inline)) {
        const uint32_t at = (uint32_t)k / 64 * F::BYTES, into = lds0 + ((uint32_t)(k - begin) / 64 & (kImages - 1)) * F::BYTES;
#pragma unroll
        for (int x = 0; x < EACH; ++x) to_lds(rsrc, into + (wave * EACH + x) * 1024, lane * 16, at + (wave * EACH + x) * 1024);
        if (REST && wave == 0) {
#pragma unroll
            for (int x = 0; x < REST; ++x) to_lds(rsrc, into + (kWaves * EACH + x) * 1024, lane * 16, at + (kWaves * EACH + x) * 1024);
        }
    };

    // rows: n of A, n of B; those past the tile's are its last
    int position[2], oldest[2], low[2], all_from[2];
    u32x4 q[2][S];
    auto window_of = [&](int p) { return a.window && p - (int64_t)a.window + 1 > INT32_MIN ? (int)(p - (int64_t)a.window + 1) : INT32_MIN; };
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int r = min(wave * 64 + b * 32 + n, t.rows - 1);
        const Row at = row_of(g, t, kv, r);
        position[b] = t.at + ((int)at.row - t.first);
        oldest[b] = window_of(position[b]);
        low[b] = __builtin_amdgcn_readlane(position[b], 0);
        all_from[b] = window_of(__builtin_amdgcn_readlane(position[b], 31));
        const T* row = (const T*)a.q + at.row * a.ldq + at.head * c.dim;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float v[8];
            u32x4 one[1];
            query<DT>(row, s * 16 + half * 8, c.dim, v);
            terms_of<1, F::QH>(v, one);
            q[b][s] = one[0];
            asm volatile("" : "+a"(q[b][s]));
        }
    }
    float R[2] = {kUnset, kUnset}, l[2] = {0.0f, 0.0f};
    f32x16 o[2][D], score[2];
    u32x4 weight[2][2], kf[S], vf[D][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[b][d][i] = 0.0f;
            asm volatile("" : "+a"(o[b][d]));
        }
        weight[b][0] = weight[b][1] = u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int d = 0; d < D; ++d) vf[d][0] = vf[d][1] = u32x4{0, 0, 0, 0};

    const uint32_t key_at = F::key_at(n, half), value_at = F::value_at(n, half), scale_at = F::SCALES + half * 16;
    auto read_key = [&](uint32_t base, int s) __attribute__((always_inline)) { kf[s] = *reinterpret_cast<const u32x4*>(lds + base + s * 32); };
    auto read_value = [&](uint32_t base, int x) __attribute__((always_inline)) {
        vf[x / 2][x % 2] = *reinterpret_cast<const u32x4*>(lds + base + x % 2 * 32 + x / 2 * 32 * F::VALUE_ROW);
    };
    // The scales of this lane's keys 8 e + 4 half .. + 3 of the 32 whose scales are at `at`.
    f32x4 sk[4], sv[4];
    auto read_scales = [&](uint32_t at, int e, f32x4& k, f32x4& v) __attribute__((always_inline)) {
        k = *reinterpret_cast<const f32x4*>(lds + at + e * 32);
        v = *reinterpret_cast<const f32x4*>(lds + at + 256 + e * 32);
    };

    // A turn: the products of rows 1 - B (scores of the keys in kf, results of the values in vf), and the weights of rows B
    // for the 32 keys from k, of which `there` are there and whose scales are at `scales`.  The first turn, B = 0, reads the next keys and values from
    // next_key and next_value on, the second one the next scales, each after its last use.
    auto turn = [&](auto rows, int k, uint32_t there, uint32_t scales, uint32_t next_key, uint32_t next_value, uint32_t next_scales) __attribute__((always_inline)) {
        constexpr int B = decltype(rows)::value, P = 1 - B;
        float p[16], sum = 0.0f;
        // largest pair of weights; of keys that some rows do not see none is right
        const int edge = (there != 0xffffffffu) | (k + 31 > low[B]) | (k < all_from[B]);
        uint32_t top = edge ? 0x8000u : 0;
        auto product = [&](int x) __attribute__((always_inline)) {
            if (x < S) scores<F::QH>(kf[x], q[P][x], score[P], x == 0);
            else results(vf[(x - S) % D][(x - S) / D], weight[P][(x - S) / D], o[P][(x - S) % D]);
        };
        const uint32_t keys = kept(next_key), values = kept(next_value), after = kept(next_scales);
        auto read = [&](int x) __attribute__((always_inline)) {
            if (B) return;
            if (x < S) read_key(keys, x);
            else read_value(values, (x - S) % D * 2 + (x - S) / D);
        };
        asm volatile("" : "+v"(score[B]));
        // an exponential between two products, and what becomes of it between the next two
        auto exponential = [&](int e) __attribute__((always_inline)) {
            p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[B][e], sk[e / 4][e % 4], -R[B]));
        };
        auto weigh = [&](int e) __attribute__((always_inline)) {
            sum = e ? sum + p[e] : p[e];
            asm volatile("" : "+v"(sum));      // here, not all of them behind the last product
            p[e] *= sv[e / 4][e % 4];
            if (e % 2) {
                const uint32_t w = halved(p[e - 1], p[e]);
                weight[B][e / 8][e / 2 % 4] = w;
                top = larger(top, w);
            }
            if (B && e % 4 == 3) read_scales(after, e / 4, sk[e / 4], sv[e / 4]);
        };
        constexpr int EACH_WEIGHTS = 16 / PRODUCTS > 1 ? 16 / PRODUCTS : 1;      // weights between two products
#pragma unroll
        for (int x = 0; x < PRODUCTS; ++x) {
            product(x);
#pragma unroll
            for (int y = 0; y < EACH_WEIGHTS; ++y) {
                if (x) weigh((x - 1) * EACH_WEIGHTS + y);
                exponential(x * EACH_WEIGHTS + y);
            }
            if (x) read(x - 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        read(PRODUCTS - 1);
#pragma unroll
        for (int y = 0; y < EACH_WEIGHTS; ++y) weigh((PRODUCTS - 1) * EACH_WEIGHTS + y);
        if (__builtin_expect(__any(too_large(top) || !(l[B] + sum <= kMostSum)), 0)) {
            uint32_t seen = 0xffff;
            if (edge) {
                // bits 8 q + 4 half + z, of keys up to this row's position and from its window's first
                const int to = position[B] < k ? 0 : min(position[B] - k + 1, 32), from = oldest[B] > k ? min(oldest[B] - k, 32) : 0;
                uint32_t mask = there & (uint32_t)((1ull << to) - 1) & ~(uint32_t)((1ull << from) - 1);
                mask >>= 4 * half;
                seen = (mask & 0xf) | (mask >> 4 & 0xf0) | (mask >> 8 & 0xf00) | (mask >> 12 & 0xf000);
            }
            const uint32_t here = kept(scales);
            Reference r(R[B], &fars[wave][B][kept((uint32_t)n)]);
            const float down = moved<32>(r, l[B], 15.0f - kRoom, [&](auto each) __attribute__((always_inline)) {
                const uint32_t mask = kept(seen);
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    f32x4 ks, vs;
                    read_scales(here, e / 4, ks, vs);
#pragma unroll
                    for (int z = 0; z < 4; ++z) each(mask >> (e + z) & 1, score[B][e + z], ks[z], vs[z]);
                    if (DP == 64 && e == 4) __builtin_amdgcn_sched_barrier(0);      // half of the scales in registers at a time
                }
            });
            R[B] = r.R;
            r.keep(&fars[wave][B][kept((uint32_t)n)]);
            if (__any(down != 1.0f)) {
                l[B] *= down;
#pragma unroll
                for (int d = 0; d < D; ++d) {
                    settled_acc(o[B][d]);
                    o[B][d] *= down;
                    asm volatile("" : "+a"(o[B][d]));
                }
            }
            auto again = [&](auto exponent_of) __attribute__((always_inline)) {
                sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    f32x4 ks, vs;
                    read_scales(here, e / 4, ks, vs);
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const bool on = seen >> (e + z) & 1;
                        p[z] = __builtin_amdgcn_exp2f(exponent_of(score[B][e + z], ks[z]));
                        p[z] = on ? p[z] : 0.0f;
                        vs[z] = on ? vs[z] : 0.0f;
                        sum += p[z];
                        p[z] *= vs[z];
                        if (z % 2) weight[B][e / 8][(e + z) / 2 % 4] = halved(p[z - 1], p[z]);
                    }
                    if (DP == 64 && e == 4) __builtin_amdgcn_sched_barrier(0);
                }
            };
            if (__builtin_expect(__any(r.is_far()), 0)) {
                const Reference wide(R[B], &fars[wave][B][kept((uint32_t)n)]);
                again([&](float t, float k) __attribute__((always_inline)) { return exponent(wide, t, k); });
            } else {
                again([&](float t, float k) __attribute__((always_inline)) { return __builtin_fmaf(t, k, -R[B]); });
            }
        }
        l[B] += sum;
    };

    // of this wave's loads all but the last `later` images' have arrived
    auto arrived = [&](auto later) __attribute__((always_inline)) {
        constexpr int N = decltype(later)::value;
        if (wave == 0) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "i"(N * (EACH + REST)) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "i"(N * EACH) : "memory");
    };
    if (begin < end) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // only images are counted from here on
        // images past the end are some that the workspace holds, or zeros past it: what is computed of them is not used
        load(begin);
        load(begin + 64);
        load(begin + 128);
        arrived(Int<2>{});
        {
            const uint32_t keys = kept(key_at);
#pragma unroll
            for (int s = 0; s < S; ++s) read_key(keys, s);
#pragma unroll
            for (int s = 0; s < S; ++s) scores<F::QH>(kf[s], q[0][s], score[0], s == 0);
        }
        settled(score[0]);
        uint32_t image = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) read_scales(scale_at, e, sk[e], sv[e]);
        uint64_t bits = *reinterpret_cast<const uint64_t*>(lds + F::SCALES + 512);
        for (int k = begin; k < end; k += 64) {
            const uint32_t next = image == (kImages - 1) * F::BYTES ? 0 : image + F::BYTES;
            const uint32_t lower = (uint32_t)__builtin_amdgcn_readfirstlane((int)bits), upper = (uint32_t)__builtin_amdgcn_readfirstlane((int)(bits >> 32));
            const uint32_t scales = image + scale_at;
            turn(Int<0>{}, k, lower, scales, image + key_at + 32 * F::KEY_ROW, image + value_at, 0);
            turn(Int<1>{}, k, lower, scales, 0, 0, scales + 128);
            // the next image is there, and all waves are done with the one before this
            arrived(Int<1>{});
            bits = *reinterpret_cast<const uint64_t*>(lds + next + F::SCALES + 512);
            load(k + 192);
            turn(Int<0>{}, k + 32, upper, scales + 128, next + key_at, image + value_at + 64, 0);
            turn(Int<1>{}, k + 32, upper, scales + 128, 0, 0, next + scale_at);
            image = next;
        }
        // the last results of B
#pragma unroll
        for (int x = 0; x < 2 * D; ++x) results(vf[x % D][x / D], weight[1][x / D], o[1][x % D]);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int d = 0; d < D; ++d) settled_acc(o[b][d]);
        l[b] += __shfl_xor(l[b], 32);
        const int r = wave * 64 + b * 32 + n;
        if (r >= t.rows) continue;
        const Row at = row_of(g, t, kv, r);
        put_row<DT, DP>(g, at, piece, pieces, half, Reference(R[b], &fars[wave][b][n]), l[b], o[b]);
    }
}

template <int DT, int DP> hipError_t run(const AttentionArgs& g, uint32_t pieces, hipStream_t s) {
    const uint32_t tiles = g.slots * g.a.at.heads;
    hipError_t e = launch(&image_kernel<DT, DP>, dim3(g.images_each * g.a.at.heads * g.a.at.seqs), 256, g, s);
    if (e == hipSuccess) e = launch(&prompt_kernel<DT, DP>, dim3(tiles, pieces), kThreads, g, s);
    if (e != hipSuccess || pieces == 1) return e;
    return launch(&join_kernel<DT, DP, kRows>, dim3(tiles, kRows * DP / 2048), 256, g, s);
}

}  // namespace

hipError_t launch_prompt(int dtype, const AttentionArgs& g, uint32_t pieces, hipStream_t s) {
    if (dtype == Q8_F16) return g.a.at.dim <= 64 ? run<Q8_F16, 64>(g, pieces, s) : run<Q8_F16, 128>(g, pieces, s);
    return g.a.at.dim <= 64 ? run<Q8_BF16, 64>(g, pieces, s) : run<Q8_BF16, 128>(g, pieces, s);
}

hipError_t prepare_prompt() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, reinterpret_cast<const void*>(&prompt_kernel<Q8_F16, 64>));
}

}  // namespace q8
