// Attention of new tokens over a paged cache of 8-bit keys and values (gfx950): what its kernels share.
//
// A tile is some rows of one sequence and one of the cache's heads; a row is a token and one of the heads
// that share it, so keys and values are read once for all of them.  Per key j and row r, with the keys' and values'
// scales sk, sv:
//     t_rj = (q_r . k_j) (sk_j scale log2 e),  p_rj = 2^(t_rj - R_r),  l_r = sum p_rj,  O_r = sum (p_rj sv_j) v_j
// over the 8-bit k_j and v_j, which 16 bits hold exactly.  R_r is no less than the largest t_rj + log2 sv_j by more
// than a fixed distance, so that p_rj sv_j fits half precision whatever the scales; it moves, and l and O with it, only
// where a product would pass 2^15, or the sum of the p_rj 2^120: those of keys with small values, or none, may be that
// large.  A scale below 2^-100 counts as that in R, and p_rj are 2^106 at most where R was just set.
// out = O / l, lse = (R + log2 l) / log2 e.
//
// The scores are taken transposed, keys by rows: a lane then has four keys of each 16 for one row, which as they
// are make the operand of the second product, O^T = V^T P^T, as the order of the keys in its sum is free.
#pragma once

#include "cache_device.hpp"

namespace q8 {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kUnset = -0x1p127f;         // R of a row that has seen no key
constexpr float kTop = 0x1p15f;             // the largest p sv
constexpr float kRoom = 6.0f;               // log2 of it where R was just set
constexpr float kLeastScale = 0x1p-100f;    // of values, as R takes them
constexpr float kWide = 0x1p24f;            // scores that leave R no room for the rest
// The largest sum of p of a lane, and how far R moves where it comes near without a p that moves R: a row's lanes and waves
// may be added, and 2^31 keys' products stay above half precision's least step.
constexpr float kMostSum = 0x1p120f, kSpare = 8.0f;

// Half precision (H) or BF16, eight values of the summed index a lane.
template <bool H> __device__ __forceinline__ void mfma16(u32x4 a, u32x4 b, f32x4& c) {
    if constexpr (H) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// 8-bit values as 16-bit ones.  Half precision: 1024 + (q + 128) is 0x6400 with q + 128 as its low byte, less 1152; BF16: the
// upper halves of the FP32 values.  `w` for half precision has its bytes' top bits turned, q + 128.
constexpr uint32_t kTurn = 0x80808080u;
__device__ __forceinline__ uint32_t halves(uint32_t w, uint32_t bytes) {     // bytes: of w, and 4 between them
    const f16x2 less = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, bytes)) + less);
}
// The four bytes of a word.
template <bool H> __device__ __forceinline__ u32x2 four(uint32_t w) {
    if constexpr (H) {
        w ^= kTurn;
        return u32x2{halves(w, 0x04010400u), halves(w, 0x04030402u)};
    } else {
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = (float)(int8_t)(w >> (8 * e));
        return u32x2{uppers(__builtin_bit_cast(uint32_t, f[0]), __builtin_bit_cast(uint32_t, f[1])),
                     uppers(__builtin_bit_cast(uint32_t, f[2]), __builtin_bit_cast(uint32_t, f[3]))};
    }
}
// Eight words turned: their first bytes, second, third and fourth ones.
template <bool H> __device__ __forceinline__ void columns(const uint32_t (&w)[8], u32x4 (&r)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t x = w[2 * e], y = w[2 * e + 1];
        if constexpr (H) {
            const uint32_t lo = __builtin_amdgcn_perm(y, x, 0x05010400u) ^ kTurn, hi = __builtin_amdgcn_perm(y, x, 0x07030602u) ^ kTurn;
            r[0][e] = halves(lo, 0x04010400u);
            r[1][e] = halves(lo, 0x04030402u);
            r[2][e] = halves(hi, 0x04010400u);
            r[3][e] = halves(hi, 0x04030402u);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float fx = (float)(int8_t)(x >> (8 * j)), fy = (float)(int8_t)(y >> (8 * j));
                r[j][e] = uppers(__builtin_bit_cast(uint32_t, fx), __builtin_bit_cast(uint32_t, fy));
            }
        }
    }
}

// Eight FP32 values as the terms of a product: one of 16 bits, rounded, or three of BF16 that hold all bits.
template <int TERMS, bool H> __device__ __forceinline__ void terms_of(const float (&v)[8], u32x4 (&t)[TERMS]) {
    if constexpr (TERMS == 1) {
        t[0] = H ? Type<Q8_F16>::eight(v) : Type<Q8_BF16>::eight(v);
    } else {
        uint32_t b[8][3];
#pragma unroll
        for (int e = 0; e < 8; ++e) three(v[e], b[e]);
#pragma unroll
        for (int n = 0; n < 3; ++n)
            t[n] = u32x4{uppers(b[0][n], b[1][n]), uppers(b[2][n], b[3][n]), uppers(b[4][n], b[5][n]), uppers(b[6][n], b[7][n])};
    }
}

// Loaded data as it is: else the compiler takes its bytes apart where it is loaded, a step early, and keeps them in
// more registers than there are.
__device__ __forceinline__ uint32_t kept(uint32_t w) {
    asm("" : "+v"(w));
    return w;
}

// A tile: rows row .. row + rows of the sequence's, and the keys that one of them sees at least.
struct Place {
    int b, first, tokens;       // sequence, its first row of the tensors, its chunk
    int row, rows;
    int at;                     // position of the chunk's first token
    int begin, end;             // keys
};
__device__ __forceinline__ int pieces_of(const Place& t, uint32_t piece) {
    return (int)(((uint32_t)max(t.end - t.begin, 0) + piece - 1) / piece);
}
// The end of the piece that begins at key `begin`: by what is left, since a window's first key and a piece as long as the table
// may pass 2^31 together.
__device__ __forceinline__ int piece_end(const Place& t, int begin, uint32_t piece) { return begin + min(t.end - begin, (int)piece); }
// The tile of slot `slot`, found by every wave for itself: tiles counted over 64 sequences at a time.
__device__ __forceinline__ bool find_tile(const AttentionArgs& g, uint32_t slot, int height, Place& t) {
    const Paged& c = g.a.at;
    const uint32_t lane = threadIdx.x & 63;
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < c.seqs; b0 += 64) {
        const uint32_t b = b0 + lane;
        int first = 0, tokens = 0, length = 0;
        if (b < c.seqs) {
            first = chunk_begin(c, b);
            tokens = max(chunk_end(c, b) - first, 0);
            length = max(c.lengths[b], 0);
        }
        const uint32_t rows = (uint32_t)tokens * g.a.group;
        const uint32_t tiles = rows > g.least && rows <= g.most ? (rows + (uint32_t)height - 1) / (uint32_t)height : 0;
        uint32_t sum = tiles;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t o = (uint32_t)__shfl_up((int)sum, d);
            if ((int)lane >= d) sum += o;
        }
        const uint64_t past = __ballot(before + sum > slot);
        if (past) {
            const int l = __builtin_ctzll(past);
            t.b = (int)b0 + l;
            t.first = __builtin_amdgcn_readlane(first, l);
            t.tokens = __builtin_amdgcn_readlane(tokens, l);
            length = __builtin_amdgcn_readlane(length, l);
            const uint32_t mine = slot - before - (uint32_t)__builtin_amdgcn_readlane((int)(sum - tiles), l);
            t.row = (int)mine * height;
            t.rows = min(height, t.tokens * (int)g.a.group - t.row);
            t.at = length - t.tokens;
            const int low = t.at + (int)divide(t.row, g.by_group), high = t.at + (int)divide(t.row + t.rows - 1, g.by_group);
            const int held = (int)min((uint32_t)length, c.width * c.page_tokens);
            t.end = min(high + 1, held);
            t.begin = g.a.window ? (int)max((int64_t)0, (int64_t)low - g.a.window + 1) : 0;
            return true;
        }
        before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
    }
    return false;
}

struct Row {
    uint64_t row, head;
};
// The tensors' row and the head of a tile's row.
__device__ __forceinline__ Row row_of(const AttentionArgs& g, const Place& t, uint32_t kv, int r) {
    const uint32_t of = (uint32_t)(t.row + r), token = divide(of, g.by_group);
    return Row{(uint64_t)(uint32_t)(t.first + (int)token), (uint64_t)(kv * g.a.group + of - token * g.a.group)};
}

// Two values for other work-groups, on any of the device's L2s, which a fence would have to write back and empty as a
// whole (0.1 us a work-group, one after the other: 8 sequences of 4096 keys 95 us, 21 without): each pair goes through to memory, and is read there.
__device__ __forceinline__ void publish(float* to, float x, float y) {
    const uint64_t w = (uint64_t)__builtin_bit_cast(uint32_t, y) << 32 | __builtin_bit_cast(uint32_t, x);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(to), w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void published(const float* from, float& x, float& y) {
    const uint64_t w = __hip_atomic_load(reinterpret_cast<const uint64_t*>(from), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    x = __builtin_bit_cast(float, (uint32_t)w);
    y = __builtin_bit_cast(float, (uint32_t)(w >> 32));
}

// A launch for the type and the values of a head.
template <typename F> hipError_t for_head(int dtype, uint32_t dim, const F& f) {
    auto held = [&](auto dt) {
        switch (held_dim(dim)) {
            case 64: return f(dt, Int<64>{});
            case 128: return f(dt, Int<128>{});
            default: return f(dt, Int<256>{});
        }
    };
    return dtype == Q8_F32 ? held(Int<Q8_F32>{}) : dtype == Q8_F16 ? held(Int<Q8_F16>{}) : held(Int<Q8_BF16>{});
}

// Eight of a row's values from d on, zeros past dim.  (Without branches: of a row's pieces, as many as DP / 8, each would
// have its own.)
template <int DT> __device__ __forceinline__ void query(const typename Type<DT>::T* row, uint32_t d, uint32_t dim, float (&v)[8]) {
    if (dim % 8 == 0) {
        Type<DT>::load8(row + (d < dim ? d : 0), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = d < dim ? v[e] : 0.0f;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = Type<DT>::get(row + min(d + e, dim - 1));
            v[e] = d + e < dim ? x : 0.0f;
        }
    }
}

// R as it moves.  Scores of 2^24 and more leave no room in FP32 for 2^15 beside them: R is then the largest score, as FP32
// holds it, and `rest` what else belongs to the reference, R + rest.  The kernels' steps know it as -infinity then: every
// exponential is infinite, or no number, and comes to where R moves, as do those of a row that has seen no key.
struct Far {
    float base, rest;           // R and what else
};
struct Reference {
    float R;                    // kUnset: no key seen; -infinity: `far` has it
    Far far;
    __device__ __forceinline__ Reference(float r, const Far* kept_far) : R(r), far{r, 0.0f} {
        if (__builtin_expect(__any(is_far()), 0) && is_far()) far = *kept_far;
    }
    __device__ __forceinline__ bool is_far() const { return R == -__builtin_huge_valf(); }
    __device__ __forceinline__ void keep(Far* kept_far) const {
        if (__builtin_expect(__any(is_far()), 0) && is_far()) *kept_far = far;
    }
};
// A score rounded, without the operation that follows.
__device__ __forceinline__ float rounded(float score, float sk) {
    float t = score * sk;
    asm("" : "+v"(t));
    return t;
}
__device__ __forceinline__ float exponent(const Reference& r, float score, float sk) {
    return r.is_far() ? (rounded(score, sk) - r.far.base) - r.far.rest : __builtin_fmaf(score, sk, -r.R);
}
__device__ __forceinline__ float log_scale(float sv) { return __builtin_amdgcn_logf(fmaxf(fabsf(sv), kLeastScale)); }
// The largest of a row's lanes, which are APART and so on to 64 apart.
template <int APART> __device__ __forceinline__ float of_row(float x) {
#pragma unroll
    for (int m = APART; m < 64; m *= 2) x = fmaxf(x, __shfl_xor(x, m));
    return x;
}
// The reference anew, the same for a row's lanes; returns the factor for their sums.  `keys` calls what it is given with each of the
// lane's keys: whether the row sees it, its score, its scales.  The reference moves where one asks for `slack` more
// than it is; l is the lane's sum.
template <int APART, typename Keys> __device__ __forceinline__ float moved(Reference& r, float l, float slack, const Keys& keys) {
    float most = kUnset;
    keys([&](bool on, float score, float sk, float sv) __attribute__((always_inline)) {
        most = on ? fmaxf(most, __builtin_fmaf(score, sk, log_scale(sv))) : most;
    });
    most = of_row<APART>(most);
    bool full = false;
    if (__builtin_expect(__any(l > 0.5f * kMostSum), 0)) full = of_row<APART>(l) > 0.5f * kMostSum;
    const float before = r.far.base;
    const float next = most > before + slack ? most - kRoom : full ? before + kSpare : before;
    float down = __builtin_amdgcn_exp2f(before - next);
    const bool wide = r.is_far() || !(fabsf(next) < kWide || next == kUnset);
    if (__builtin_expect(__any(wide), 0)) {
        float top = kUnset, want = kUnset;
        keys([&](bool on, float score, float sk, float) __attribute__((always_inline)) { top = on ? fmaxf(top, rounded(score, sk)) : top; });
        const float base = fmaxf(before, of_row<APART>(top)), old = (before - base) + r.far.rest;
        keys([&](bool on, float score, float sk, float sv) __attribute__((always_inline)) {
            want = on ? fmaxf(want, (rounded(score, sk) - base) + log_scale(sv)) : want;
        });
        want = of_row<APART>(want) - kRoom;
        const float rest = want > old + (slack - kRoom) ? want : full ? old + kSpare : old;
        if (wide) {
            down = 1.0f;
            if (rest > old || base != before) {
                const bool fits = fabsf(base) < kWide;
                const Far now = fits ? Far{base + rest, 0.0f} : Far{base, rest};
                down = __builtin_amdgcn_exp2f((before - now.base) + (r.far.rest - now.rest));
                r.R = fits ? now.base : -__builtin_huge_valf();
                r.far = now;
            }
            return down;
        }
    }
    r.R = next;
    return down;
}
// Sums whose reference is R alone: the factor for O.  The p then are 2^(t - R), R the largest t or so.
__device__ __forceinline__ float without_rest(const Reference& r, float& R, float& l) {
    R = r.far.base;
    const float up = __builtin_amdgcn_exp2f(r.far.rest);
    l *= up;
    return up;
}
// A piece's sums, so that those of thousands of pieces can be added: the factor for O.
__device__ __forceinline__ float settle(float& R, float& l) {
    const bool large = l > 0x1p64f;
    R += large ? 32.0f : 0.0f;
    const float down = large ? 0x1p-32f : 1.0f;
    l *= down;
    return down;
}

// Sums of some keys with those of others.
__device__ __forceinline__ void add_part(float& R, float& l, float (&v)[8], float r, float lr, const float (&o)[8]) {
    const float next = fmaxf(R, r), down = __builtin_amdgcn_exp2f(R - next), part = __builtin_amdgcn_exp2f(r - next);
    R = next;
    l = l * down + lr * part;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * down + o[e] * part;
}

}  // namespace q8
