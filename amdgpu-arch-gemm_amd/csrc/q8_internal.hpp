// Interface between the 8-bit operators' host code (q8_shim.cpp) and their
// kernels (q8_rows.hip, q8_pack.hip, q8_gemm.hip).  Nothing here is part of
// the C-ABI.
#pragma once

#include "q8_shim.h"

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

#define Q8_INTERNAL __attribute__((visibility("hidden")))

namespace q8 {

inline uint32_t type_bytes(int dtype) { return dtype == Q8_F32 ? 4u : 2u; }
inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// Rows of `cols` values at `ld` elements.
struct Quantize {
    const void* x;
    int8_t* q;
    float* scale;
    uint32_t ldx, ldq, rows, cols;
    // the norm's (residual, hidden, rstd may be null)
    const void* residual;
    const void* gain;
    void* hidden;
    float* rstd;
    uint32_t ldr, ldh;
    float eps;
};
Q8_INTERNAL hipError_t launch_quantize(int dtype, bool norm, const Quantize& p, hipStream_t stream);

struct Dequantize {
    const int8_t* q;
    const float* scale;
    void* y;
    uint32_t ldq, ldy, rows, cols;
};
Q8_INTERNAL hipError_t launch_dequantize(int dtype, const Dequantize& p, hipStream_t stream);

struct NormBackward {
    const void* dn;
    const void* hidden;
    const void* gain;
    const float* rstd;
    const void* dres;     // may be null
    void* dx;
    float* dgain;         // may be null
    float* partial;       // parts x cols, where dgain is wanted
    uint32_t lddn, ldh, lddr, lddx, rows, cols, parts;
};
// Row ranges that the gain's gradient is summed over first.
Q8_INTERNAL uint32_t norm_backward_parts(uint32_t rows);
Q8_INTERNAL hipError_t launch_norm_backward(int dtype, const NormBackward& p, hipStream_t stream);

// What the matrix cores multiply.
enum Element { E_I8 = 0, E_F16 = 1, E_BF16 = 2 };

// One product D = A B^T: rows of A and of B hold the summed index, `kb` bytes of it.
struct Product {
    const void* a;
    const void* b;
    uint64_t lda, ldb;    // bytes
    uint32_t m, n, kb;
    const float* sx;      // E_I8: scales of A's and B's rows
    const float* sw;
    const void* bias;     // E_I8: of type `out`, may be null
    const float* alpha;   // E_F16: a factor in device memory; null: 1
    void* y;
    uint64_t ldy;         // elements
    int out;
    int accumulate;
    // set by the launcher
    uint32_t nwgx, nwgy, splits, tiles_per_split;
    uint32_t rows, pitch; // of a K range's sums: whole tiles
    // by the caller: splits sums of whole tiles, where the route has more than one
    void* partial;
};

// How a product runs: `kind` of q8_plan.hpp, and the K ranges.
struct Route {
    int kind;
    uint32_t splits;
};
Q8_INTERNAL hipError_t launch_product(Element e, const Route& r, const Product& p, hipStream_t stream);
Q8_INTERNAL hipError_t launch_direct(const Product& p, hipStream_t stream);   // E_I8, rows that start anywhere
// Each kernel source is a code object of its own, which its prepare function loads on the current device.
Q8_INTERNAL hipError_t prepare_products();
Q8_INTERNAL hipError_t prepare_rows();
Q8_INTERNAL hipError_t prepare_packing();
Q8_INTERNAL hipError_t prepare_gradients();
Q8_INTERNAL hipError_t prepare_cache_rows();
Q8_INTERNAL hipError_t prepare_few();
Q8_INTERNAL hipError_t prepare_many();
Q8_INTERNAL hipError_t prepare_prompt();

// 8-bit rows to rows of whole 16 bytes: dst[r][0 .. cols) and zeros up to dst_ld.
Q8_INTERNAL hipError_t launch_copy_rows(const int8_t* src, uint64_t src_ld, int8_t* dst, uint64_t dst_ld, uint32_t rows,
                                        uint32_t cols, hipStream_t stream);
// The two operands of a gradient, laid out with the summed index along the rows, `cp` values of
// it (a multiple of eight; zeros past the `rows` or `cols` of the source).
//   weights:  dst[j][t * cp + c] = scale_c q_cj, rounded to 16 bits; with scale == null (F32)
//             q_cj alone, `terms` times.  F16: times pair[0] = 2^-e, and pair[1] = 2^e, such that
//             the largest finite scale * 2^-e is in [2^7, 2^8); both are set here.
//   gradient: dst[i][t * cp + c] = term t of src_ic (transposed: src_ci).  16-bit types: one term,
//             copied; F32: scaled by scale_c, three BF16 terms.
// dst_ld and src_ld in elements.
struct PackWeights {
    const int8_t* q;
    const float* scale;
    float* pair;
    void* dst;
    uint64_t ldq, dst_ld;
    uint32_t rows, cols, cp, terms;
};
struct PackGradient {
    const void* src;
    const float* scale;
    void* dst;
    uint64_t src_ld, dst_ld;
    uint32_t rows, cols, cp;  // rows: of dst; cols: values of the summed index
    int transposed;
};
// gradient: null where it is read as it is.
Q8_INTERNAL hipError_t launch_pack(int dtype, const PackWeights& weights, const PackGradient* gradient, hipStream_t stream);

// A gradient from operands as they are: d[r][c] = sum over s of a_r,s scale_s q_s,c (turned: a_s,r), of
// type `out`, Q8_F32 or a's.  cols >= 4; turned: rows >= 8, else sum >= 32; F16: sum <= kFewScales.
struct Gradient {
    const void* a;
    const int8_t* q;
    const float* scale;
    void* d;
    uint64_t lda, ldq, ldd;
    uint32_t rows, cols, sum;
    int out, accumulate;
};
Q8_INTERNAL hipError_t launch_gradient(int dtype, bool turned, const Gradient& p, hipStream_t stream);

}  // namespace q8
