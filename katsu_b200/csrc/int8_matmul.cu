// y = (x in 8 bits) (w in 8 bits) with a scale for each token and channel: entry points, and the product for many tokens.
#include "int8.cuh"

namespace {

int32_t check(const int8_t *wq, const float *ws, const float *y, size_t m, size_t k, size_t n) {
    KATSU_REQUIRE(k >= 1 && k <= KATSU_INT8_MAX_K, "k must be 1 to KATSU_INT8_MAX_K");
    KATSU_REQUIRE(m <= 0x3fffffff && n <= 0x3fffffff, "too many rows or columns");
    if (m == 0 || n == 0) return KATSU_OK;
    KATSU_REQUIRE(wq != nullptr && ws != nullptr && y != nullptr, "null buffer");
    KATSU_REQUIRE((reinterpret_cast<uintptr_t>(wq) & 15u) == 0, "a quantised matrix must be 16-byte aligned");
    return KATSU_OK;
}

int32_t product(katsu_cuda_ctx *ctx, const int8_t *xq, const float *xs, const int8_t *wq, const float *ws, const float *bias,
                float *y, size_t m, size_t k, size_t n) {
    const size_t pitch = katsu_int8_pitch(k);
    size_t step = 8;
    while (step * pitch > size_t(200) * 1024) step /= 2;
    for (size_t i = 0; i < m; i += step) {
        int handled = 0;
        const size_t rows = m - i < step ? m - i : step;
        KATSU_TRY(katsu_int8_few(ctx, nullptr, xq + i * pitch, xs + i, wq, ws, bias, y + i * n, rows, k, n, &handled));
    }
    return KATSU_OK;
}

}  // namespace

extern "C" int32_t katsu_cuda_int8_matmul(katsu_cuda_ctx *ctx, const int8_t *xq, const float *xs, const int8_t *wq,
                                          const float *ws, const float *bias, float *y, size_t m, size_t k, size_t n) {
    KATSU_REQUIRE(ctx != nullptr, "null context");
    KATSU_TRY(check(wq, ws, y, m, k, n));
    if (m == 0 || n == 0) return katsu_bind(ctx);
    KATSU_REQUIRE(xq != nullptr && xs != nullptr, "null buffer");
    for (const void *in : {(const void *)xq, (const void *)xs, (const void *)wq, (const void *)ws, (const void *)bias})
        KATSU_REQUIRE(in != y, "y is an input too");
    KATSU_REQUIRE((reinterpret_cast<uintptr_t>(xq) & 15u) == 0, "a quantised matrix must be 16-byte aligned");
    KATSU_TRY(katsu_bind(ctx));
    return product(ctx, xq, xs, wq, ws, bias, y, m, k, n);
}

extern "C" int32_t katsu_cuda_int8_linear(katsu_cuda_ctx *ctx, const float *x, const int8_t *wq, const float *ws,
                                          const float *bias, float *y, size_t m, size_t k, size_t n) {
    KATSU_REQUIRE(ctx != nullptr, "null context");
    KATSU_TRY(check(wq, ws, y, m, k, n));
    if (m == 0 || n == 0) return katsu_bind(ctx);
    KATSU_REQUIRE(x != nullptr, "null buffer");
    for (const void *in : {(const void *)x, (const void *)wq, (const void *)ws, (const void *)bias})
        KATSU_REQUIRE(in != y, "y is an input too");
    KATSU_TRY(katsu_bind(ctx));
    int handled = 0;
    KATSU_TRY(katsu_int8_few(ctx, x, nullptr, nullptr, wq, ws, bias, y, m, k, n, &handled));
    if (handled) return KATSU_OK;
    const size_t pitch = katsu_int8_pitch(k), scales = katsu_div_up(m, 64) * 64;
    float *scratch = nullptr;
    KATSU_TRY(katsu_scratch(ctx, scales + katsu_div_up(m * pitch, 4), &scratch));
    int8_t *xq = reinterpret_cast<int8_t *>(scratch + scales);
    KATSU_TRY(katsu_int8_quantize(ctx, x, xq, scratch, m, k));
    return product(ctx, xq, scratch, wq, ws, bias, y, m, k, n);
}
