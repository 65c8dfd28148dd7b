// Host side of the 8-bit operators (include/q8_shim.h): handles, argument checks,
// workspace, and which kernels a call runs on.
#include "cache_plan.hpp"
#include "q8_host.hpp"
#include "q8_plan.hpp"

#include <cstdint>
#include <new>

namespace {

using namespace q8;

// As plan_grad, refusing a sum that is too long.
int plan(int dtype, bool turned, bool odd, uint64_t rows, uint64_t cols, uint64_t sum, bool copy_a, GradPlan& g) {
    const bool f32 = dtype == Q8_F32;
    const uint64_t most = most_summed(grad_terms(f32));
    if (sum > most)
        return fail(SGEMM_E_SHAPE, "a sum over %llu products is too long: at most %llu", (unsigned long long)sum,
                    (unsigned long long)most);
    g = plan_grad(f32, dtype == Q8_F16, turned, odd, rows, cols, sum, copy_a);
    return SGEMM_OK;
}

int check_grid(uint64_t m, uint64_t n, const ProductPlan& p) {
    const Tile& t = kTiles[p.kind];
    // 2^32 work-items are one grid's end
    if (div_up(m, t.m) * div_up(n, t.n) >= (1u << 22))
        return fail(SGEMM_E_SHAPE, "%llu x %llu outputs are more tiles than a grid holds", (unsigned long long)m,
                    (unsigned long long)n);
    return SGEMM_OK;
}

bool rows_aligned(const void* p, uint64_t ld_bytes) {
    return (uintptr_t)p % 16 == 0 && ld_bytes % 16 == 0 && ld_bytes <= kMaxRowBytes;
}

bool odd_rows(const void* p, uint64_t ld_bytes) { return ((uintptr_t)p | ld_bytes) % 4 != 0; }

void set_common(Product& p, q8_handle* h, const ProductPlan& plan, const Layout& at) {
    p.partial = plan.partial_bytes ? h->workspace + at.partial : nullptr;
}

}  // namespace

extern "C" {

int q8_open(q8_handle** out) {
    if (!out) return fail(SGEMM_E_INVALID, "out is null");
    *out = nullptr;
    int count = 0;
    if (hipGetDeviceCount(&count) != hipSuccess || count < 1) return fail(SGEMM_E_NO_DEVICE, "no HIP device is visible");
    q8_handle* h = new (std::nothrow) q8_handle;
    if (!h) return fail(SGEMM_E_INVALID, "out of host memory");
    const BesideCaptures beside;
    hipError_t e = hipGetDevice(&h->device);
    if (e == hipSuccess) e = hipStreamCreate(&h->own_stream);
    // no call loads code: a first one may be under capture, and should not take longer than the next
    if (e == hipSuccess) e = prepare_rows();
    if (e == hipSuccess) e = prepare_packing();
    if (e == hipSuccess) e = prepare_products();
    if (e == hipSuccess) e = prepare_gradients();
    if (e == hipSuccess) e = prepare_cache_rows();
    if (e == hipSuccess) e = prepare_few();
    if (e == hipSuccess) e = prepare_many();
    if (e == hipSuccess) e = prepare_prompt();
    if (e == hipSuccess) e = hipMalloc(reinterpret_cast<void**>(&h->tickets), kTickets * sizeof(uint32_t));
    if (e == hipSuccess) e = hipMemsetAsync(h->tickets, 0, kTickets * sizeof(uint32_t), h->own_stream);
    if (e == hipSuccess) e = hipStreamSynchronize(h->own_stream);
    if (e != hipSuccess) {
        if (h->tickets) (void)hipFree(h->tickets);
        if (h->own_stream) (void)hipStreamDestroy(h->own_stream);
        delete h;
        return hip_fail(e, "q8_open");
    }
    h->stream = h->own_stream;
    *out = h;
    return SGEMM_OK;
}

void q8_close(q8_handle* h) {
    if (!h) return;
    OnDevice on(h->device);
    (void)hipStreamSynchronize(h->stream);
    if (h->workspace) (void)hipFree(h->workspace);
    while (h->retired) {
        q8_handle::Retired* r = h->retired;
        h->retired = r->next;
        (void)hipFree(r->memory);
        delete r;
    }
    if (h->tickets) (void)hipFree(h->tickets);
    if (h->own_stream) (void)hipStreamDestroy(h->own_stream);
    delete h;
}

int q8_set_stream(q8_handle* h, void* stream) {
    CHECK(check_handle(h));
    OnDevice on(h->device);
    HIP_TRY(on.status());
    hipStream_t next = stream ? static_cast<hipStream_t>(stream) : h->own_stream;
    if (next == h->stream) return SGEMM_OK;
    if (stream) {
        int device = 0;
        HIP_TRY(hipStreamGetDevice(next, &device));
        if (device != h->device)
            return fail(SGEMM_E_INVALID, "the stream belongs to device %d, the handle to %d", device, h->device);
    }
    if (capturing(h->stream)) return fail(SGEMM_E_INVALID, "the handle's stream is capturing");
    HIP_TRY(hipStreamSynchronize(h->stream));
    h->stream = next;
    return SGEMM_OK;
}

int q8_synchronize(q8_handle* h) {
    CHECK(check_handle(h));
    HIP_TRY(hipStreamSynchronize(h->stream));
    return SGEMM_OK;
}

int q8_reserve(q8_handle* h, size_t bytes) {
    CHECK(check_handle(h));
    OnDevice on(h->device);
    HIP_TRY(on.status());
    return grow(h, bytes);
}

int q8_workspace_size(int call, int dtype, uint32_t m, uint32_t n, uint32_t k, size_t* bytes) {
    if (!bytes) return fail(SGEMM_E_INVALID, "bytes is null");
    *bytes = 0;
    CHECK(check_type(dtype));
    if (call == Q8_CALL_RMSNORM_BACKWARD) {
        *bytes = Layout::piece((size_t)norm_backward_parts(m) * k * sizeof(float));
    } else if (call == Q8_CALL_GEMM) {
        for (int copies = 0; copies < 4; ++copies) {    // the route depends on them
            const size_t need = plan_gemm(m, n, k, copies & 1, copies & 2).at.total;
            if (need > *bytes) *bytes = need;
        }
    } else if (call == Q8_CALL_GRAD_INPUT || call == Q8_CALL_GRAD_WEIGHT) {
        for (int i = 0; i < 4; ++i) {   // the route depends on dy's rows
            GradPlan g;
            if (call == Q8_CALL_GRAD_INPUT) CHECK(plan(dtype, false, i & 2, m, k, n, i & 1, g));
            else CHECK(plan(dtype, true, i & 2, n, k, m, true, g));
            if (g.at.total > *bytes) *bytes = g.at.total;
        }
    } else {
        return fail(SGEMM_E_INVALID, "%d is no call with a workspace", call);
    }
    return SGEMM_OK;
}

int q8_quantize(q8_handle* h, int dtype, const void* x, uint32_t ldx, int8_t* q, uint32_t ldq, float* scale,
                uint32_t rows, uint32_t cols) {
    CHECK(check_handle(h));
    CHECK(check_type(dtype));
    if (!rows) return SGEMM_OK;
    if (!cols) return fail(SGEMM_E_SHAPE, "rows of no values have no scale");
    const Span sx{"x", x, rows, cols, ldx, type_bytes(dtype)}, sq{"q", q, rows, cols, ldq, 1}, ss = vec("scale", scale, rows, 4);
    CHECK(check(sx));
    CHECK(check(sq));
    CHECK(check(ss));
    CHECK(check_apart(sq, sx));
    CHECK(check_apart(ss, sx));
    CHECK(check_apart(ss, sq));
    OnDevice on(h->device);
    HIP_TRY(on.status());
    Quantize p = {};
    p.x = x; p.q = q; p.scale = scale; p.ldx = ldx; p.ldq = ldq; p.rows = rows; p.cols = cols;
    return launched(launch_quantize(dtype, false, p, h->stream), "launch of the quantisation failed");
}

int q8_dequantize(q8_handle* h, int dtype, const int8_t* q, uint32_t ldq, const float* scale, void* y, uint32_t ldy,
                  uint32_t rows, uint32_t cols) {
    CHECK(check_handle(h));
    CHECK(check_type(dtype));
    if (!rows || !cols) return SGEMM_OK;
    const Span sq{"q", q, rows, cols, ldq, 1}, ss = vec("scale", scale, rows, 4), sy{"y", y, rows, cols, ldy, type_bytes(dtype)};
    CHECK(check(sq));
    CHECK(check(ss));
    CHECK(check(sy));
    CHECK(check_apart(sy, sq));
    CHECK(check_apart(sy, ss));
    OnDevice on(h->device);
    HIP_TRY(on.status());
    const Dequantize p = {q, scale, y, ldq, ldy, rows, cols};
    return launched(launch_dequantize(dtype, p, h->stream), "launch of the restoring failed");
}

int q8_rmsnorm(q8_handle* h, int dtype, const void* x, uint32_t ldx, const void* residual, uint32_t ldr,
               const void* gain, void* hidden, uint32_t ldh, int8_t* q, uint32_t ldq, float* scale, float* rstd,
               uint32_t rows, uint32_t cols, float eps) {
    CHECK(check_handle(h));
    CHECK(check_type(dtype));
    if (!(eps >= 0.0f && eps <= 3.4e38f)) return fail(SGEMM_E_INVALID, "eps is negative or no number");
    if (!rows) return SGEMM_OK;
    if (!cols) return fail(SGEMM_E_SHAPE, "rows of no values have no norm");
    const uint32_t size = type_bytes(dtype);
    const Span in[] = {{"x", x, rows, cols, ldx, size}, {"residual", residual, residual ? rows : 0u, cols, ldr, size},
                       vec("gain", gain, cols, size)};
    const Span out[] = {{"hidden", hidden, hidden ? rows : 0u, cols, ldh, size}, {"q", q, rows, cols, ldq, 1},
                        vec("scale", scale, rows, 4), vec("rstd", rstd, rstd ? rows : 0u, 4)};
    for (const Span& s : in) CHECK(check(s));
    for (const Span& s : out) CHECK(check(s));
    for (int i = 0; i < 4; ++i) {
        for (int j = 0; j < 3; ++j) CHECK(check_apart(out[i], in[j], i == 0 && j < 2));
        for (int j = 0; j < i; ++j) CHECK(check_apart(out[i], out[j]));
    }
    OnDevice on(h->device);
    HIP_TRY(on.status());
    const Quantize p = {x, q, scale, ldx, ldq, rows, cols, residual, gain, hidden, rstd, ldr, ldh, eps};
    return launched(launch_quantize(dtype, true, p, h->stream), "launch of the norm failed");
}

int q8_rmsnorm_backward(q8_handle* h, int dtype, const void* dn, uint32_t lddn, const void* hidden, uint32_t ldh,
                        const void* gain, const float* rstd, const void* dres, uint32_t lddr, void* dx, uint32_t lddx,
                        float* dgain, uint32_t rows, uint32_t cols) {
    CHECK(check_handle(h));
    CHECK(check_type(dtype));
    if (!cols) return SGEMM_OK;
    const uint32_t size = type_bytes(dtype);
    const Span in[] = {{"dn", dn, rows, cols, lddn, size}, {"hidden", hidden, rows, cols, ldh, size},
                       vec("gain", gain, cols, size), vec("rstd", rstd, rows, 4),
                       {"dres", dres, dres ? rows : 0u, cols, lddr, size}};
    const Span out[] = {{"dx", dx, rows, cols, lddx, size}, vec("dgain", dgain, dgain ? cols : 0u, 4)};
    for (const Span& s : in) CHECK(check(s));
    for (const Span& s : out) CHECK(check(s));
    for (int j = 0; j < 5; ++j) {
        CHECK(check_apart(out[0], in[j], j == 0 || j == 4));
        CHECK(check_apart(out[1], in[j]));
    }
    CHECK(check_apart(out[0], out[1]));
    if (!rows && !dgain) return SGEMM_OK;
    OnDevice on(h->device);
    HIP_TRY(on.status());
    NormBackward p = {dn, hidden, gain, rstd, dres, dx, dgain, nullptr, lddn, ldh, lddr, lddx, rows, cols,
                      norm_backward_parts(rows)};
    if (dgain && rows) {
        CHECK(take_workspace(h, (size_t)p.parts * cols * sizeof(float)));
        p.partial = reinterpret_cast<float*>(h->workspace);
    }
    return launched(launch_norm_backward(dtype, p, h->stream), "launch of the norm's gradient failed");
}

int q8_gemm(q8_handle* h, int dtype, const int8_t* qx, uint32_t ldx, const float* sx, const int8_t* qw, uint32_t ldw,
            const float* sw, const void* bias, void* y, uint32_t ldy, uint32_t m, uint32_t n, uint32_t k) {
    CHECK(check_handle(h));
    CHECK(check_type(dtype));
    if (!m || !n) return SGEMM_OK;
    if (k > Q8_MAX_K) return fail(SGEMM_E_SHAPE, "k = %u: sums of more than %u products may not fit 32 bits", k, Q8_MAX_K);
    const uint32_t size = type_bytes(dtype);
    const Span in[] = {{"qx", qx, m, k, ldx, 1}, {"qw", qw, n, k, ldw, 1}, vec("sx", sx, m, 4), vec("sw", sw, n, 4),
                       vec("bias", bias, bias ? n : 0u, size)};
    const Span out{"y", y, m, n, ldy, size};
    for (const Span& s : in) CHECK(check(s));
    CHECK(check(out));
    for (const Span& s : in) CHECK(check_apart(out, s));
    // a sum that ends inside a piece of 16 bytes: qx's copy has zeros there, and what qw has
    // is multiplied by them
    const GemmPlan g = plan_gemm(m, n, k, !rows_aligned(qx, ldx) || k % 16, !rows_aligned(qw, ldw));
    if (!g.direct) CHECK(check_grid(m, n, g.plan));
    else if (n >= (1u << 28)) return fail(SGEMM_E_SHAPE, "%u channels are more than a grid holds", n);
    OnDevice on(h->device);
    HIP_TRY(on.status());
    CHECK(take_workspace(h, g.at.total));
    Product p = {};
    p.a = qx; p.b = qw; p.lda = ldx; p.ldb = ldw; p.m = m; p.n = n; p.kb = k;
    p.sx = sx; p.sw = sw; p.bias = bias; p.y = y; p.ldy = ldy; p.out = dtype;
    if (g.direct) return launched(launch_direct(p, h->stream), "launch of the product failed");
    if (g.copy_a) {
        p.a = h->workspace + g.at.a;
        p.lda = g.ldc;
        HIP_TRY(launch_copy_rows(qx, ldx, reinterpret_cast<int8_t*>(h->workspace + g.at.a), g.ldc, m, k, h->stream));
    }
    if (g.copy_b) {
        p.b = h->workspace + g.at.b;
        p.ldb = g.ldc;
        HIP_TRY(launch_copy_rows(qw, ldw, reinterpret_cast<int8_t*>(h->workspace + g.at.b), g.ldc, n, k, h->stream));
    }
    set_common(p, h, g.plan, g.at);
    return launched(launch_product(E_I8, Route{g.plan.kind, g.plan.splits}, p, h->stream), "launch of the product failed");
}

int q8_grad_input(q8_handle* h, int dtype, const void* dy, uint32_t lddy, const int8_t* qw, uint32_t ldw,
                  const float* sw, void* dx, uint32_t lddx, uint32_t m, uint32_t n, uint32_t k) {
    CHECK(check_handle(h));
    CHECK(check_type(dtype));
    if (!m || !k) return SGEMM_OK;
    const uint32_t size = type_bytes(dtype);
    const Span in[] = {{"dy", dy, m, n, lddy, size}, {"qw", qw, n, k, ldw, 1}, vec("sw", sw, n, 4)};
    const Span out{"dx", dx, m, k, lddx, size};
    // dy's rows hold the summed index: read where they are if they are whole pieces
    const bool copy = dtype == Q8_F32 || n % 8 || !rows_aligned(dy, (uint64_t)lddy * size);
    GradPlan g;
    CHECK(plan(dtype, false, odd_rows(dy, (uint64_t)lddy * size), m, k, n, copy, g));
    if (!g.direct) CHECK(check_grid(m, k, g.plan));
    for (const Span& s : in) CHECK(check(s));
    CHECK(check(out));
    for (const Span& s : in) CHECK(check_apart(out, s));
    OnDevice on(h->device);
    HIP_TRY(on.status());
    if (g.direct) {
        const Gradient p = {dy, qw, sw, dx, lddy, ldw, lddx, m, k, n, dtype, 0};
        return launched(launch_gradient(dtype, false, p, h->stream), "launch of the input's gradient failed");
    }
    CHECK(take_workspace(h, g.at.total));
    const Element e = dtype == Q8_F16 ? E_F16 : E_BF16;
    float* pair = dtype == Q8_F16 ? reinterpret_cast<float*>(h->workspace + g.at.pair) : nullptr;
    if (n) {
        const PackWeights pw = {qw, dtype == Q8_F32 ? nullptr : sw, pair, h->workspace + g.at.b, ldw, g.pitch / 2, n, k,
                                (uint32_t)g.cp, g.terms};
        const PackGradient pg = {dy, dtype == Q8_F32 ? sw : nullptr, h->workspace + g.at.a, lddy, g.pitch / 2, m, n,
                                 (uint32_t)g.cp, 0};
        HIP_TRY(launch_pack(dtype, pw, copy ? &pg : nullptr, h->stream));
    } else {
        pair = nullptr;
    }
    Product p = {};
    p.a = copy ? h->workspace + g.at.a : dy;
    p.lda = copy ? g.pitch : (uint64_t)lddy * size;
    p.b = h->workspace + g.at.b;
    p.ldb = g.pitch;
    p.m = m; p.n = k; p.kb = (uint32_t)g.kb;
    p.alpha = pair; p.y = dx; p.ldy = lddx; p.out = dtype;
    set_common(p, h, g.plan, g.at);
    return launched(launch_product(e, Route{g.plan.kind, g.plan.splits}, p, h->stream), "launch of the input's gradient failed");
}

int q8_grad_weight(q8_handle* h, int dtype, const void* dy, uint32_t lddy, const int8_t* qx, uint32_t ldx,
                   const float* sx, int out_dtype, void* dw, uint32_t lddw, uint32_t m, uint32_t n, uint32_t k,
                   int accumulate) {
    CHECK(check_handle(h));
    CHECK(check_type(dtype));
    if (out_dtype != dtype && out_dtype != Q8_F32)
        return fail(SGEMM_E_INVALID, "dw's type %d is neither dy's (%d) nor Q8_F32", out_dtype, dtype);
    if (!n || !k || (!m && accumulate)) return SGEMM_OK;
    const uint32_t size = type_bytes(dtype);
    const Span in[] = {{"dy", dy, m, n, lddy, size}, {"qx", qx, m, k, ldx, 1}, vec("sx", sx, m, 4)};
    const Span out{"dw", dw, n, k, lddw, type_bytes(out_dtype)};
    GradPlan g;
    CHECK(plan(dtype, true, odd_rows(dy, (uint64_t)lddy * size), n, k, m, true, g));
    if (!g.direct) CHECK(check_grid(n, k, g.plan));
    for (const Span& s : in) CHECK(check(s));
    CHECK(check(out));
    for (const Span& s : in) CHECK(check_apart(out, s));
    OnDevice on(h->device);
    HIP_TRY(on.status());
    if (g.direct) {
        const Gradient p = {dy, qx, sx, dw, lddy, ldx, lddw, n, k, m, out_dtype, accumulate != 0};
        return launched(launch_gradient(dtype, true, p, h->stream), "launch of the weights' gradient failed");
    }
    CHECK(take_workspace(h, g.at.total));
    const Element e = dtype == Q8_F16 ? E_F16 : E_BF16;
    float* pair = dtype == Q8_F16 ? reinterpret_cast<float*>(h->workspace + g.at.pair) : nullptr;
    if (m) {
        const PackWeights pw = {qx, dtype == Q8_F32 ? nullptr : sx, pair, h->workspace + g.at.b, ldx, g.pitch / 2, m, k,
                                (uint32_t)g.cp, g.terms};
        const PackGradient pg = {dy, dtype == Q8_F32 ? sx : nullptr, h->workspace + g.at.a, lddy, g.pitch / 2, n, m,
                                 (uint32_t)g.cp, 1};
        HIP_TRY(launch_pack(dtype, pw, &pg, h->stream));
    } else {
        pair = nullptr;
    }
    Product p = {};
    p.a = h->workspace + g.at.a;
    p.b = h->workspace + g.at.b;
    p.lda = p.ldb = g.pitch;
    p.m = n; p.n = k; p.kb = (uint32_t)g.kb;
    p.alpha = pair; p.y = dw; p.ldy = lddw; p.out = out_dtype; p.accumulate = accumulate != 0;
    set_common(p, h, g.plan, g.at);
    return launched(launch_product(e, Route{g.plan.kind, g.plan.splits}, p, h->stream),
                    "launch of the weights' gradient failed");
}

}  // extern "C"
