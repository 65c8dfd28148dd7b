// Products of the 8-bit operators on the matrix cores (gfx950).
//
// product_kernel: D = A B^T for rows that hold the summed index, in 8-bit
// integers (int32 sums, exact) or 16-bit floats (FP32 sums).  All three have operands of 16
// bytes a lane and rows of 128 bytes a K tile, so one kernel serves them:
//   memory --buffer_load ... lds, 16 bytes a lane--> LDS, two or three buffers --> MFMA
// finish_kernel adds the sums of K ranges where a product has too few tiles.
// direct_kernel: few tokens and small products; operands go from memory to the matrix cores.
//
// What bounds the large products.  8192^3 in 8-bit integers takes 405 - 433 us by card, 2.5 - 2.7 Pops (a
// large library product 2.35); 16384 x 4096 x 4096 in BF16 400 - 415 us, 1.33 - 1.37 PFLOP/s (library 1.32).
// The card's power (a loop of matrix instructions alone reaches 4.0 Pops and 2.0 PFLOP/s on such data;
// here the clock falls from 2.4 to 1.8 and 1.9 GHz, and the matrix instructions are busy 64% and 66 - 72% of the cycles),
// and the loads' way into LDS: without any load 375 us instead of 430, in BF16
// 362 instead of 413.  Not memory: with every load from lines that L2 holds the times are the same.
// Four waves of 128 x 128 rather than eight of 128 x 64: LDS gives 128 bytes a cycle, and eight
// waves would ask it for 192 KB a K tile beside the 64 KB that arrive, as long as the matrix
// instructions take (the step from eight to four: 4096^3 74.0 -> 57.5 us, 8192^3 464 -> 453).
#include "q8_device.hpp"
#include "q8_internal.hpp"
#include "q8_plan.hpp"

namespace q8 {
namespace {

constexpr int BUFFER_RSRC_WORD3 = 0x00020000;
constexpr uint32_t NOWHERE = 0x80000000u;    // an offset past every descriptor's end: loads give 0
constexpr int KB = kTileBytes;

// The matrix instructions: `in_place` keeps a sum in its registers (the compiler else copies
// between the two halves of the register file, up to an instruction for each of them), and its
// user waits for the results.
template <int E> struct Atom;
template <> struct Atom<E_I8> {
    typedef i32x4 Acc;
    static __device__ __forceinline__ void mfma(u32x4 a, u32x4 b, Acc& c) {
        c = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
    }
    template <bool AGPR> static __device__ __forceinline__ void in_place(u32x4 a, u32x4 b, Acc& c) {
        if constexpr (AGPR) asm("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
        else asm("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
    }
};
template <> struct Atom<E_F16> {
    typedef f32x4 Acc;
    template <bool AGPR> static __device__ __forceinline__ void in_place(u32x4 a, u32x4 b, Acc& c) {
        if constexpr (AGPR) asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
        else asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
    }
};
template <> struct Atom<E_BF16> {
    typedef f32x4 Acc;
    template <bool AGPR> static __device__ __forceinline__ void in_place(u32x4 a, u32x4 b, Acc& c) {
        if constexpr (AGPR) asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
        else asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
    }
};

// Tiles in groups of six rows of them, column by column within a group: the 32 tiles of
// 256 x 256 that an XCD works on at a time are then 6 x 5.3 and read the fewest
// lines.  With `ask` below it matters little: 8192^3 in 8-bit integers takes 426 - 436 us with three to
// eight, 444 with sixteen; F16 4096 x 4096 x 16384 390 - 396 and 403.
__device__ __forceinline__ void tile_of(uint32_t z, uint32_t nx, uint32_t ny, uint32_t& tx, uint32_t& ty) {
    constexpr uint32_t GROUP = 6;
    const uint32_t group = z / (GROUP * ny), first = group * GROUP;
    const uint32_t width = min(nx - first, GROUP), in = z - group * GROUP * ny;
    tx = first + in % width;
    ty = in / width;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* base, uint64_t ld, uint32_t row0, uint32_t rows,
                                                            uint32_t kb) {
    // a last piece of less than 16 bytes is read whole: it starts at a multiple of 16,
    // so the bytes past the matrix lie in the same page
    const uint64_t left = (uint64_t)(rows - 1 - row0) * ld + ((kb + 15u) & ~15u);
    return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)base + (uint64_t)row0 * ld), (short)0,
                                             (int)(left < 0x7fffffffu ? left : 0x7fffffffu), BUFFER_RSRC_WORD3);
}

// 1024 bytes, 16 a lane, to LDS from `lds` + at on; soff then moves on by `step`.  The
// assembly form, since the compiler would wait for it before every read of LDS; the
// barrier of the next K tile waits.  (m0 needs no clobber: it is reserved, and set
// right before each use; the addition between the two is the wait state it needs.)
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t rsrc, uint32_t lds, int at, uint32_t voff, uint32_t& soff,
                                         uint32_t step) {
    uint32_t from;
    asm volatile("s_add_u32 m0, %2, %6\n\ts_mov_b32 %0, %1\n\ts_add_u32 %1, %1, %5\n\tbuffer_load_dwordx4 %3, %4, %0 offen lds"
                 : "=&s"(from), "+s"(soff) : "s"(lds), "v"(voff), "s"(rsrc), "s"(step), "i"(at) : "scc");
}

// One dword a lane, 256 bytes of LDS.
__device__ __forceinline__ void touch(__amdgpu_buffer_rsrc_t rsrc, uint32_t lds, uint32_t voff, uint32_t soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
                 :: "s"(lds), "v"(voff), "s"(rsrc), "s"(soff));
}

// Waits for the wave's reads of LDS, which the compiler then knows (lgkmcnt 0).
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(0xc07f); }

template <bool V> struct Flag { static constexpr bool value = V; };
template <int V> struct Int { static constexpr int value = V; };

__device__ __forceinline__ float out_value(int v) { return (float)v; }
__device__ __forceinline__ float out_value(float v) { return v; }

// 2 x 2 waves of T x T tiles of 16 x 16: 256 x 256 outputs with T = 8, one wave a SIMD,
// or 128 x 128 with T = 4, two work-groups a CU.
//
// A K tile is two steps of 64 bytes.  While one step is multiplied, the next one's
// operands are read from LDS between the matrix instructions; a tile's buffer is
// free once its second step has been read, in the middle of the tile, and takes the
// tile after next then.  So there is one barrier a tile, and a load has the time of a whole
// tile to land.  AHEAD: see `ask`.  DT: D's type.  NBUF: buffers; with more than two the loads
// are as many tiles further ahead.
template <int E, int DT, int T, int NBUF, bool AHEAD>
__global__ void __launch_bounds__(256, T == 4 ? 2 : 1) product_kernel(const Product p) {
    typedef Atom<E> A;
    typedef typename A::Acc Acc;
    constexpr int TM = T, TN = T, WAVES = 4, BM = 2 * T * 16, BN = BM;
    constexpr int LOADS = BM / 8 / WAVES;                       // of 8 rows a wave, K tile and operand
    constexpr int STAGE = (BM + BN) * KB;
    constexpr int LDS = NBUF * STAGE + (AHEAD ? WAVES * 256 : 0);
    __shared__ __attribute__((aligned(128))) unsigned char lds[LDS];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave & 1, wn = wave >> 1;
    uint32_t tx, ty;
    tile_of(xcd_order(blockIdx.x, p.nwgx * p.nwgy), p.nwgx, p.nwgy, tx, ty);
    const uint32_t row0 = tx * BM, col0 = ty * BN;
    const uint32_t tiles_k = (p.kb + KB - 1) / KB;
    const uint32_t k_first = blockIdx.y * p.tiles_per_split;
    const uint32_t k_last = min(k_first + p.tiles_per_split, tiles_k);

    const __amdgpu_buffer_rsrc_t ra = rows_rsrc(p.a, p.lda, row0, p.m, p.kb), rb = rows_rsrc(p.b, p.ldb, col0, p.n, p.kb);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;

    // Row r of a tile keeps its piece c of 16 bytes at piece c ^ key(r), so that the lanes that
    // read LDS together meet all banks: rows fr of A, and those of B that `read` says.
    // A load's lanes fill LDS in order, so it is the address in memory that is permuted.
    const uint32_t lr = (uint32_t)lane >> 3;
    const uint32_t ca = ((uint32_t)lane & 7u) ^ lr, cb = ((uint32_t)lane & 7u) ^ ((lr & 3u) | ((uint32_t)wave & 1u) << 2);
    const uint32_t lda = (uint32_t)p.lda, ldb = (uint32_t)p.ldb;
    const uint32_t va = (uint32_t)(wave * 8 + lr) * lda + ca * 16u, vb = (uint32_t)(wave * 8 + lr) * ldb + cb * 16u;
    const uint32_t stepa = WAVES * 8u * lda, stepb = WAVES * 8u * ldb;
    // past which byte of a row nothing is read: pieces from there on are zeros
    const uint32_t k_end = min(k_last * KB, p.kb);
    uint32_t ua = 0, ub = 0, sa = 0, sb = 0, at = 0;    // of the tile that is being loaded
    auto aim = [&](uint32_t kt, uint32_t buf) __attribute__((always_inline)) {
        sa = sb = kt * KB;
        ua = sa + ca * 16u < k_end ? va : NOWHERE;
        ub = sa + cb * 16u < k_end ? vb : NOWHERE;
        at = lds0 + buf * STAGE + (uint32_t)wave * 1024u;
    };
    auto load = [&](int i) __attribute__((always_inline)) {     // 0 .. 2 * LOADS - 1, A and B in turn
        const int r = i / 2 * (WAVES * 1024);
        if (i & 1) load_lds(rb, at, BM * KB + r, ub, sb, stepb);
        else load_lds(ra, at, r, ua, sa, stepa);
    };

    // A tile's loads have the time of one tile, which L2 keeps and memory does not: a dword of
    // each of its lines is asked for one tile before, into LDS that nobody reads.  The
    // work-groups beside this one on the XCD share its rows of A or of B, so each
    // asks for a quarter of them (F16 4096 x 4096 x 16384: 405 -> 393 us, 8192^3 in 8-bit integers
    // 438 -> 431, BF16 16384 x 4096 x 4096 415 -> 413).
    constexpr uint32_t SHARE = BM / 4;
    const uint32_t pr = (wave < 2 ? ty % 4 : tx % 4) * SHARE + (uint32_t)(wave & 1) * (SHARE / 2) + (uint32_t)lane;
    const uint32_t pp = (uint32_t)lane < SHARE / 2 ? pr * (wave < 2 ? lda : ldb) : NOWHERE;
    auto ask = [&](uint32_t kt) __attribute__((always_inline)) {
        const uint32_t v = kt < k_last ? pp : NOWHERE;
        if (wave < 2) touch(ra, lds0 + NBUF * STAGE + (uint32_t)wave * 256u, v, kt * KB);
        else touch(rb, lds0 + NBUF * STAGE + (uint32_t)wave * 256u, v, kt * KB);
    };

    Acc acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = Acc{0, 0, 0, 0};

    // The wave's operands: a lane has row fr of a tile of A, and of a tile of B the row with
    // which its results are columns next to one another: in a pair of tiles, row fr of tile j
    // is row fr / 4 * 8 + j * 4 + fr % 4, and a lane's eight results are columns fg * 8 .. + 7.
    const uint32_t fr = (uint32_t)lane & 15u, fg = (uint32_t)lane >> 4;
    const uint32_t fa = (uint32_t)(wm * TM * 16) * KB + fr * KB + (fg ^ (fr & 7u)) * 16u;
    const uint32_t fb = (uint32_t)(BM + wn * TN * 16) * KB + ((fr >> 2) * 8u + (fr & 3u)) * KB +
                        (fg ^ ((fr & 3u) | ((fr >> 2) & 1u) << 2)) * 16u;
    struct Step {
        u32x4 a[TM], b[TN];
    };
    Step f0, f1;
    auto read = [&](Step& f, uint32_t buf, uint32_t s, int i) __attribute__((always_inline)) {   // 0 .. TM + TN - 1
        const unsigned char* from = lds + buf * STAGE;
        if (i < TN) f.b[i] = *reinterpret_cast<const u32x4*>(from + (fb ^ (s * 64)) + (i / 2 * 32 + i % 2 * 4) * KB);
        else f.a[i - TN] = *reinterpret_cast<const u32x4*>(from + (fa ^ (s * 64)) + (i - TN) * 16 * KB);
    };
    // One step's products, the next step's operands and, in the second step, a tile's loads
    // between them, evenly: all at its start make 431 us 461 (8192^3 in 8-bit integers).
    auto multiply = [&](const Step& f, Step& next, uint32_t buf, uint32_t s, auto loads) __attribute__((always_inline)) {
        constexpr int N = TM * TN, GAP = N / (TM + TN) - 1, EVERY = N / (2 * LOADS);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int x = i * TN + j;
                if (x % GAP == 0 && x / GAP < TM + TN) read(next, buf, s, x / GAP);
                if (decltype(loads)::value && x % EVERY == EVERY - 1) load(x / EVERY);
                A::template in_place<T == 8>(f.b[j], f.a[i], acc[i][j]);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    if (k_first < k_last) {
#pragma unroll
        for (int b = 0; b < NBUF; ++b) {
            aim(k_first + b, b);
#pragma unroll
            for (int i = 0; i < 2 * LOADS; ++i) load(i);
        }
        if constexpr (AHEAD) ask(k_first + NBUF);
        constexpr int LATER = 2 * LOADS * (NBUF - 2) + (AHEAD ? 1 : 0);     // loads that a tile's barrier leaves
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "i"(2 * LOADS + LATER) : "memory");
#pragma unroll
        for (int i = 0; i < TM + TN; ++i) read(f0, 0, 0, i);
        wait_lds();
        uint32_t buf = 0;
        for (uint32_t kt = k_first; kt < k_last; ++kt) {
            const uint32_t next = buf + 1 == NBUF ? 0 : buf + 1;
            multiply(f0, f1, buf, 1, Flag<false>{});
            // every wave has read this tile, and the next one has landed
            wait_lds();
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" :: "i"(LATER) : "memory");
            aim(kt + NBUF, buf);
            multiply(f1, f0, next, 0, Flag<true>{});
            if constexpr (AHEAD) ask(kt + NBUF + 1);
            wait_lds();
            buf = next;
        }
        // zeros for tiles past the range; and the last products, whose results the
        // compiler does not know to wait for
        asm volatile("s_waitcnt vmcnt(0)\n\ts_nop 15\n\ts_nop 15" ::: "memory");
    }
    // A sum, read no earlier than here: not before the wait above, and not all of them at once.
    auto sum = [&](int i, int j) __attribute__((always_inline)) {
        if constexpr (T == 8) asm volatile("" : "+a"(acc[i][j]));
        else asm volatile("" : "+v"(acc[i][j]));
        return acc[i][j];
    };

    const uint32_t wrow = row0 + (uint32_t)(wm * TM * 16), wcol = col0 + (uint32_t)(wn * TN * 16);
    if (p.splits > 1) {
        // a K range's sums, whole tiles: finish_kernel adds the ranges
        char* first = (char*)p.partial + (((uint64_t)blockIdx.y * p.rows + wrow + fr) * p.pitch + wcol + fg * 8u) * 4u;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                *reinterpret_cast<Acc*>(first + (uint64_t)i * 64u * p.pitch + (j / 2 * 32 + j % 2 * 4) * 4) = sum(i, j);
        return;
    }
    // D: a lane has eight columns of a row in a pair of tiles, four lanes 32.  Each wave turns 16
    // rows of 64 columns at a time in its own part of LDS, where the tiles were, and stores
    // whole rows, eight lanes each.  All scales are loaded before the first of them.
    constexpr int PITCH = 64 + 4;
    static_assert(WAVES * 16 * PITCH * 4 <= LDS, "D's rows are staged where the tiles were");
    typedef typename Type<DT>::T Out;
    const uint32_t lrow = (uint32_t)lane / 8u, lcol = (uint32_t)lane % 8u * 8u;
    float sx[TM][2], sw[TN / 4][8], bias[TN / 4][8];
    if constexpr (E == E_I8) {
#pragma unroll
        for (int h = 0; h < TN / 4; ++h) {
            const uint32_t col = wcol + h * 64u + lcol;
#pragma unroll
            for (int e = 0; e < 8; ++e) bias[h][e] = 0.0f;
            if (col < p.n) {
                load_part<Q8_F32>(p.sw, col, p.n, sw[h]);
                if (p.bias) load_part<DT>((const Out*)p.bias, col, p.n, bias[h]);
            }
        }
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int q = 0; q < 2; ++q) sx[i][q] = p.sx[min(wrow + i * 16u + q * 8u + lrow, p.m - 1)];
    }
    const float factor = E == E_F16 && p.alpha ? p.alpha[1] : 1.0f;
    __syncthreads();
    float* const stage = reinterpret_cast<float*>(lds) + wave * 16 * PITCH;
#pragma unroll
    for (int h = 0; h < TN / 4; ++h) {
        const uint32_t col = wcol + h * 64u + lcol;
        const bool on = col < p.n;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const Acc x = sum(i, 4 * h + j);
                *reinterpret_cast<f32x4*>(stage + fr * PITCH + j / 2 * 32 + fg * 8u + j % 2 * 4) =
                    f32x4{out_value(x[0]), out_value(x[1]), out_value(x[2]), out_value(x[3])};
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const uint32_t r = q * 8u + lrow, row = wrow + i * 16u + r;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const f32x4 w = *reinterpret_cast<const f32x4*>(stage + r * PITCH + lcol + e);
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[e + k] = w[k];
                }
                if (!on || row >= p.m) continue;
                Out* y = (Out*)p.y + (uint64_t)row * p.ldy;
                if constexpr (E == E_I8) {
                    finish(v, sx[i][q], sw[h], bias[h]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] *= factor;
                }
                if (E != E_I8 && p.accumulate) {
                    float old[8];
                    load_part<DT>(y, col, p.n, old);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += old[e];
                }
                store_part<DT>(y, col, p.n, v);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// The K ranges' sums of a product, added in range order and finished as the product kernel finishes
// its own: a work-group has 8 rows of 256 columns, a thread eight columns.
template <int E, int DT> __global__ void __launch_bounds__(256) finish_kernel(const Product p) {
    typedef typename Atom<E>::Acc Acc;
    typedef typename Type<DT>::T Out;
    const uint32_t blocks = (p.n + 255) / 256;
    const uint32_t row = blockIdx.x / blocks * 8 + threadIdx.x / 32, col = blockIdx.x % blocks * 256 + threadIdx.x % 32 * 8;
    if (row >= p.m || col >= p.n) return;
    const uint64_t range = (uint64_t)p.rows * p.pitch;
    const Acc* from = reinterpret_cast<const Acc*>((const char*)p.partial + ((uint64_t)row * p.pitch + col) * 4);
    Acc lo = from[0], hi = from[1];
#pragma unroll 4
    for (uint32_t s = 1; s < p.splits; ++s) {
        from += range / 4;
        lo += from[0];
        hi += from[1];
    }
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = out_value(lo[e]); v[4 + e] = out_value(hi[e]); }
    Out* y = (Out*)p.y + (uint64_t)row * p.ldy;
    float add[8] = {};
    if constexpr (E == E_I8) {
        float sw[8];
        load_part<Q8_F32>(p.sw, col, p.n, sw);
        if (p.bias) load_part<DT>((const Out*)p.bias, col, p.n, add);
        finish(v, p.sx[row], sw, add);
    } else {
        const float factor = E == E_F16 && p.alpha ? p.alpha[1] : 1.0f;
        if (p.accumulate) load_part<DT>(y, col, p.n, add);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] * factor + add[e];
    }
    store_part<DT>(y, col, p.n, v);
}

// Few tokens, or a small product (direct_kind).  A work-group owns 16 * NT channels, 16 * MT tokens and all of K, in
// runs of four steps of 64 bytes that its waves take in turn; operands go from memory
// straight to the matrix cores, from rows that start anywhere, with a run's loads in flight
// while the one before is multiplied.  The waves' sums meet in LDS.
// ODD: rows start between dwords.  Loads of 16 bytes from there take more than twice the time (1 x 2551 x
// 10881: 22.8 us, rows of 10884 9.5), so the dwords around them are read and shifted.
template <int MT, int NT, int WAVES, int DT, bool ODD>
__global__ void __launch_bounds__(WAVES * 64) direct_kernel(const Product p) {
    constexpr int RUN = ODD && MT * NT > 1 ? 2 : 4;
    typedef typename Raw<ODD>::T Piece;
    typedef Atom<E_I8> A;
    typedef typename Type<DT>::T Out;
    __shared__ __attribute__((aligned(16))) i32x4 red[WAVES][MT * NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int fr = lane & 15, fg = lane >> 4;
    const uint32_t col0 = blockIdx.x * (16 * NT), row0 = blockIdx.y * (16 * MT);
    const uint32_t whole = p.kb / 64;             // steps without an end inside
    const char* w[NT];
    const char* x[MT];
    bool wok[NT], xok[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const uint32_t c = col0 + (uint32_t)(j * 16 + fr);
        wok[j] = c < p.n;
        w[j] = (const char*)p.b + (uint64_t)(wok[j] ? c : 0u) * p.ldb + fg * 16;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const uint32_t r = row0 + (uint32_t)(i * 16 + fr);
        xok[i] = r < p.m;
        x[i] = (const char*)p.a + (uint64_t)(xok[i] ? r : 0u) * p.lda + fg * 16;
    }
    i32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    struct Run {
        Piece w[RUN][NT], x[RUN][MT];
    };
    uint32_t wat[NT], xat[MT];      // the rows' first bytes in a dword
#pragma unroll
    for (int j = 0; j < NT; ++j) wat[j] = (uint32_t)(uintptr_t)w[j] & 3u;
#pragma unroll
    for (int i = 0; i < MT; ++i) xat[i] = (uint32_t)(uintptr_t)x[i] & 3u;
    const u32x4 zero = {0, 0, 0, 0};
    auto fetch = [&](Run& v, uint32_t s0) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < RUN; ++s) {
            const uint64_t at = (uint64_t)(s0 + s) * 64;
            const bool on = s0 + s < whole;
#pragma unroll
            for (int j = 0; j < NT; ++j) v.w[s][j] = on && wok[j] ? Raw<ODD>::load(w[j] + at) : Piece{};
#pragma unroll
            for (int i = 0; i < MT; ++i) v.x[s][i] = on && xok[i] ? Raw<ODD>::load(x[i] + at) : Piece{};
        }
    };
    auto multiply = [&](const Run& v) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < RUN; ++s) {
            u32x4 wv[NT], xv[MT];
#pragma unroll
            for (int j = 0; j < NT; ++j) wv[j] = Raw<ODD>::value(v.w[s][j], wat[j]);
#pragma unroll
            for (int i = 0; i < MT; ++i) xv[i] = Raw<ODD>::value(v.x[s][i], xat[i]);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) A::mfma(wv[j], xv[i], acc[i][j]);
        }
    };
    constexpr uint32_t STRIDE = WAVES * RUN;
    Run v0, v1;
    uint32_t s0 = (uint32_t)wave * RUN;
    if (s0 < whole) fetch(v0, s0);
    for (; s0 < whole; s0 += 2 * STRIDE) {
        fetch(v1, s0 + STRIDE);     // nothing past the rows' end
        multiply(v0);
        fetch(v0, s0 + 2 * STRIDE);
        multiply(v1);
    }
    if (p.kb % 64 && wave == WAVES - 1) {   // the rest, byte by byte
        const uint32_t k0 = whole * 64 + fg * 16;
        u32x4 wv[NT], xv[MT];
        auto bytes = [&](const char* s, bool ok) __attribute__((always_inline)) {
            u32x4 v = zero;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (ok && k0 + e < p.kb) v[e / 4] |= (uint32_t)(uint8_t)s[(uint64_t)whole * 64 + e] << (8 * (e % 4));
            return v;
        };
#pragma unroll
        for (int j = 0; j < NT; ++j) wv[j] = bytes(w[j], wok[j]);
#pragma unroll
        for (int i = 0; i < MT; ++i) xv[i] = bytes(x[i], xok[i]);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) A::mfma(wv[j], xv[i], acc[i][j]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) red[wave][i * NT + j][lane] = acc[i][j];
    // the scales, before the wait for the other waves
    const int t0 = wave;
    float sx = 0.0f, sw[4] = {}, bias[4] = {};
    auto aim = [&](int t) __attribute__((always_inline)) {
        const uint32_t row = row0 + (uint32_t)(t / NT * 16 + fr), col = col0 + (uint32_t)(t % NT * 16 + fg * 4);
        if (row >= p.m) return;
        sx = p.sx[row];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < p.n) {
                sw[e] = p.sw[col + e];
                if (p.bias) bias[e] = Type<DT>::get((const Out*)p.bias + col + e);
            }
    };
    if (t0 < MT * NT) aim(t0);
    __syncthreads();
    for (int t = t0; t < MT * NT; t += WAVES) {
        if (t != t0) aim(t);
        i32x4 v = red[0][t][lane];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) v += red[k][t][lane];
        const uint32_t row = row0 + (uint32_t)(t / NT * 16 + fr), col = col0 + (uint32_t)(t % NT * 16 + fg * 4);
        if (row >= p.m) continue;
        Out* y = (Out*)p.y + row * p.ldy + col;
        float r[4] = {(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
        finish(r, sx, sw, bias);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < p.n) Type<DT>::put(y + e, r[e]);
    }
}

hipError_t launch(const void* f, dim3 grid, uint32_t threads, const Product& p, hipStream_t stream) {
    void* args[] = {const_cast<Product*>(&p)};
    return hipLaunchKernel(f, grid, dim3(threads), args, 0, stream);
}

template <int E, int DT> hipError_t product_any(const Route& r, Product p, hipStream_t s) {
    const Tile& t = kTiles[r.kind];
    p.nwgx = (uint32_t)ceil_div(p.m, t.m);
    p.nwgy = (uint32_t)ceil_div(p.n, t.n);
    p.rows = p.nwgx * t.m;
    p.pitch = p.nwgy * t.n;
    const uint32_t tiles_k = (uint32_t)ceil_div(p.kb, KB);
    p.tiles_per_split = (uint32_t)tiles_per_split(p.kb, r.splits);
    p.splits = tiles_k ? (uint32_t)ceil_div(tiles_k, p.tiles_per_split) : 1;    // none is empty
    const bool ahead = asks_ahead((uint64_t)p.nwgx * p.nwgy * p.splits, p.tiles_per_split);
    const void* f = r.kind == K_SMALL        ? (const void*)&product_kernel<E, DT, 4, 2, false>
                    : r.kind == K_SMALL_DEEP ? (const void*)&product_kernel<E, DT, 4, 3, false>
                    : ahead                  ? (const void*)&product_kernel<E, DT, 8, 2, true>
                                             : (const void*)&product_kernel<E, DT, 8, 2, false>;
    const hipError_t e = launch(f, dim3(p.nwgx * p.nwgy, p.splits), 256, p, s);
    if (e != hipSuccess || p.splits == 1) return e;
    return launch((const void*)&finish_kernel<E, DT>, dim3((uint32_t)(ceil_div(p.m, 8) * ceil_div(p.n, 256))), 256, p, s);
}

template <int MT, int NT, int WAVES, bool ODD> const void* direct_of(int out) {
    return out == Q8_F32   ? (const void*)&direct_kernel<MT, NT, WAVES, Q8_F32, ODD>
           : out == Q8_F16 ? (const void*)&direct_kernel<MT, NT, WAVES, Q8_F16, ODD>
                           : (const void*)&direct_kernel<MT, NT, WAVES, Q8_BF16, ODD>;
}
template <int MT, int NT, int WAVES> hipError_t direct_any(const Product& p, hipStream_t s) {
    const bool odd = ((uintptr_t)p.a | (uintptr_t)p.b | p.lda | p.ldb) % 4 != 0;
    const void* f = odd ? direct_of<MT, NT, WAVES, true>(p.out) : direct_of<MT, NT, WAVES, false>(p.out);
    return launch(f, dim3((uint32_t)ceil_div(p.n, 16 * NT), (uint32_t)ceil_div(p.m, 16 * MT)), WAVES * 64, p, s);
}

}  // namespace

hipError_t launch_product(Element e, const Route& r, const Product& p, hipStream_t s) {
    if (e == E_F16)
        return p.out == Q8_F32 ? product_any<E_F16, Q8_F32>(r, p, s) : product_any<E_F16, Q8_F16>(r, p, s);
    if (e == E_BF16)
        return p.out == Q8_F32 ? product_any<E_BF16, Q8_F32>(r, p, s) : product_any<E_BF16, Q8_BF16>(r, p, s);
    return p.out == Q8_F32 ? product_any<E_I8, Q8_F32>(r, p, s)
                           : p.out == Q8_F16 ? product_any<E_I8, Q8_F16>(r, p, s) : product_any<E_I8, Q8_BF16>(r, p, s);
}

hipError_t launch_direct(const Product& p, hipStream_t s) {
    switch (direct_kind(p.m, p.n, p.kb)) {
        case D_1x1_16: return direct_any<1, 1, 16>(p, s);
        case D_1x1_8: return direct_any<1, 1, 8>(p, s);
        case D_1x4_8: return direct_any<1, 4, 8>(p, s);
        case D_2x1_8: return direct_any<2, 1, 8>(p, s);
        case D_2x4_8: return direct_any<2, 4, 8>(p, s);
        case D_2x2_8: return direct_any<2, 2, 8>(p, s);
        case D_4x4_4: return direct_any<4, 4, 4>(p, s);
    }
    return hipErrorInvalidValue;
}

hipError_t prepare_products() {
    hipFuncAttributes a;
    return hipFuncGetAttributes(&a, (const void*)&product_kernel<E_I8, Q8_BF16, 8, 2, false>);
}

}  // namespace q8
