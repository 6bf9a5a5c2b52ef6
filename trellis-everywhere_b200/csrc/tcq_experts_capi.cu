// C ABI of products with an epilogue, grouped products, routing and combining (declared in include/tcq_b200.h): argument checks.
#include "../../include/tcq_b200.h"

#include "tcq_experts.cuh"
#include "tcq_microscale_grouped.cuh"

using namespace tcq;

namespace {

bool misaligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }
bool bad_type(int dtype) { return dtype < TCQ_F32 || dtype > TCQ_BF16; }
size_t type_bytes(int dtype) { return dtype == TCQ_F32 ? 4 : 2; }
constexpr int64_t kMostRows = int64_t(1) << 30;          // grids, coordinates and counts of tiles fit 32 bits
constexpr int64_t kMostColumns = int64_t(1) << 24;

int check_epilogue(int64_t n, const void* bias, int bias_dtype, int activation, const void* residual, int64_t ldr, const void* y, int y_dtype, int64_t ldy) {
    if (bad_type(y_dtype) || (bias != nullptr && bad_type(bias_dtype))) return TCQ_E_BAD_FORMAT;
    if (activation < TCQ_ACT_NONE || activation > TCQ_ACT_SWIGLU || (act_gated(activation) && n % 2)) return TCQ_E_BAD_ARGUMENT;
    const int64_t out = act_gated(activation) ? n / 2 : n;
    if (ldy < out || (residual != nullptr && ldr < out)) return TCQ_E_BAD_ARGUMENT;
    if (y == nullptr) return TCQ_E_NULL_POINTER;
    if (misaligned(y, type_bytes(y_dtype)) || misaligned(residual, type_bytes(y_dtype)) || (bias != nullptr && misaligned(bias, type_bytes(bias_dtype)))) return TCQ_E_MISALIGNED;
    return TCQ_OK;
}

int check_grouped(int64_t rows, int64_t groups, int64_t n, int64_t k, int dtype, int format) {
    if (format != TCQ_MS_MXFP4 && format != TCQ_MS_NVFP4) return TCQ_E_BAD_FORMAT;
    if (dtype != TCQ_F16 && dtype != TCQ_BF16) return TCQ_E_BAD_FORMAT;
    if (rows < 0 || n < 0 || k < 0 || groups < 0) return TCQ_E_BAD_COUNT;
    if (groups < 1 || groups > kMostGroups || rows > kMostRows || n > kMostRows || k > kMostColumns || n * groups >= int64_t(1) << 31) return TCQ_E_BAD_ARGUMENT;
    // items of 128 rows of a matrix x one row of x, the most there may be
    return ((n + 127) / 128) * (rows + groups) >= int64_t(1) << 31 ? TCQ_E_BAD_ARGUMENT : TCQ_OK;
}

int grouped_core(const void* x, int dtype, int64_t x_rows, int64_t ldx, const int32_t* tokens, const int32_t* offsets, int64_t groups, int64_t rows, const uint8_t* codes,
                 const uint8_t* scales, const float* row_scale, int64_t n, int64_t k, int format, const void* bias, int bias_dtype, int activation, const void* residual,
                 int64_t ldr, void* y, int y_dtype, int64_t ldy, void* ws, size_t ws_bytes, unsigned loads, void* stream) {
    int rc = check_grouped(rows, groups, n, k, dtype, format);
    if (rc != TCQ_OK) return rc;
    if (x_rows < 0) return TCQ_E_BAD_COUNT;
    if (offsets == nullptr && groups != 1) return TCQ_E_NULL_POINTER;
    if (rows == 0 || n == 0) return TCQ_OK;
    if (k == 0 || ldx < k || x_rows >= int64_t(1) << 31 || (tokens == nullptr && x_rows < rows)) return TCQ_E_BAD_ARGUMENT;
    if ((rc = check_epilogue(n, bias, bias_dtype, activation, residual, ldr, y, y_dtype, ldy)) != TCQ_OK) return rc;
    if ((x == nullptr && x_rows > 0) || codes == nullptr || scales == nullptr || (format == TCQ_MS_NVFP4) != (row_scale != nullptr)) return TCQ_E_NULL_POINTER;
    if (misaligned(x, 2) || misaligned(codes, 16) || misaligned(scales, 16) || misaligned(row_scale, 4) || misaligned(tokens, 4) || misaligned(offsets, 4) || misaligned(ws, 256))
        return TCQ_E_MISALIGNED;
    const size_t need = ms_grouped_workspace_bytes(rows, groups, n, k, dtype, format, tokens == nullptr && ms_rows_aligned(x, ldx));
    if (need && ws == nullptr) return TCQ_E_NULL_POINTER;
    if (ws_bytes < need) return TCQ_E_WORKSPACE;
    const GroupedCall c{x, dtype, x_rows, ldx, tokens, {offsets, int(groups), int(rows)}, {codes, scales, row_scale, n}, k, format,
                        {bias, bias_dtype, activation, residual, ldr, y, y_dtype, ldy}, loads};
    const cudaError_t err = launch_ms_grouped(c, ws, static_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? TCQ_OK : report_cuda_error(err, "ms_grouped_linear");
}

}  // namespace

extern "C" {

size_t tcq_ms_grouped_linear_workspace_bytes(int64_t rows, int64_t groups, int64_t n, int64_t k, int dtype, int format, int in_order) {
    if (check_grouped(rows, groups, n, k, dtype, format) != TCQ_OK || rows == 0) return 0;
    return ms_grouped_workspace_bytes(rows, groups, n, k, dtype, format, in_order != 0);
}

int tcq_ms_grouped_linear(const void* x, int dtype, int64_t x_rows, int64_t ldx, const int32_t* tokens, const int32_t* offsets, int64_t groups, int64_t rows,
                          const uint8_t* codes, const uint8_t* scales, const float* row_scale, int64_t n, int64_t k, int format, const void* bias, int bias_dtype,
                          int activation, const void* residual, int64_t ldr, void* y, int y_dtype, int64_t ldy, void* ws, size_t ws_bytes, void* stream) {
    return grouped_core(x, dtype, x_rows, ldx, tokens, offsets, groups, rows, codes, scales, row_scale, n, k, format, bias, bias_dtype, activation, residual, ldr, y, y_dtype,
                        ldy, ws, ws_bytes, kMsAllLoads, stream);
}

int tcq_selftest_ms_grouped_waits(int64_t loads, const void* x, int dtype, int64_t x_rows, int64_t ldx, const int32_t* tokens, const int32_t* offsets, int64_t groups,
                                  int64_t rows, const uint8_t* codes, const uint8_t* scales, const float* row_scale, int64_t n, int64_t k, int format, const void* bias,
                                  int bias_dtype, int activation, const void* residual, int64_t ldr, void* y, int y_dtype, int64_t ldy, void* ws, size_t ws_bytes, void* stream) {
    if (loads < 0 || loads >= int64_t(kMsAllLoads)) return TCQ_E_BAD_COUNT;
    return grouped_core(x, dtype, x_rows, ldx, tokens, offsets, groups, rows, codes, scales, row_scale, n, k, format, bias, bias_dtype, activation, residual, ldr, y, y_dtype,
                        ldy, ws, ws_bytes, unsigned(loads), stream);
}

int tcq_ms_epilogue(const float* h, int64_t rows, int64_t n, const void* bias, int bias_dtype, int activation, const void* residual, int64_t ldr, void* y, int y_dtype,
                    int64_t ldy, void* stream) {
    if (rows < 0 || n < 0) return TCQ_E_BAD_COUNT;
    if (rows > kMostRows || n > kMostRows || rows * ((n + 3) / 4) > (int64_t(1) << 31) * 255) return TCQ_E_BAD_ARGUMENT;
    if (rows == 0 || n == 0) return TCQ_OK;
    const int rc = check_epilogue(n, bias, bias_dtype, activation, residual, ldr, y, y_dtype, ldy);
    if (rc != TCQ_OK) return rc;
    if (h == nullptr) return TCQ_E_NULL_POINTER;
    if (misaligned(h, 4)) return TCQ_E_MISALIGNED;
    const cudaError_t err = launch_epilogue(h, rows, n, {bias, bias_dtype, activation, residual, ldr, y, y_dtype, ldy}, static_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? TCQ_OK : report_cuda_error(err, "ms_epilogue");
}

size_t tcq_route_workspace_bytes(int64_t tokens, int64_t experts) {
    if (tokens <= 0 || experts <= 0 || tokens >= int64_t(1) << 31 || experts > kMostExperts) return 0;
    const int chunks = route_chunks(int(tokens));
    return chunks == 1 ? 0 : size_t(chunks) * size_t(experts) * 4;
}

int tcq_route(const void* logits, int dtype, int64_t tokens, int64_t ld, int64_t experts, int64_t top, int score, int normalize, float* weights, int32_t* chosen, int32_t* places,
              int32_t* order, int32_t* offsets, void* ws, size_t ws_bytes, void* stream) {
    if (bad_type(dtype)) return TCQ_E_BAD_FORMAT;
    if (tokens < 0) return TCQ_E_BAD_COUNT;
    if (experts < 1 || experts > kMostExperts || top < 1 || top > kMostChosen || top > experts || tokens >= (int64_t(1) << 31) / top || ld < experts ||
        (score != TCQ_SCORE_SOFTMAX && score != TCQ_SCORE_SIGMOID) || (normalize != 0 && normalize != 1))
        return TCQ_E_BAD_ARGUMENT;
    const size_t need = tcq_route_workspace_bytes(tokens, experts);
    if (offsets == nullptr || (tokens > 0 && (logits == nullptr || weights == nullptr || chosen == nullptr || places == nullptr || order == nullptr)) || (need && ws == nullptr))
        return TCQ_E_NULL_POINTER;
    if (misaligned(logits, type_bytes(dtype)) || misaligned(weights, 4) || misaligned(chosen, 4) || misaligned(places, 4) || misaligned(order, 4) || misaligned(offsets, 4) ||
        misaligned(ws, 4))
        return TCQ_E_MISALIGNED;
    if (ws_bytes < need) return TCQ_E_WORKSPACE;
    const RouteCall c{logits, dtype, ld, int(tokens), int(experts), int(top), score, normalize != 0, weights, chosen, places, order, offsets, static_cast<int*>(ws)};
    const cudaError_t err = launch_route(c, static_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? TCQ_OK : report_cuda_error(err, "route");
}

int tcq_combine(const void* y, int dtype, int64_t rows, int64_t ldy, int64_t n, const float* weights, const int32_t* places, int64_t tokens, int64_t top, const void* residual,
                int64_t ldr, void* out, int out_dtype, int64_t ldo, void* stream) {
    if (bad_type(dtype) || bad_type(out_dtype)) return TCQ_E_BAD_FORMAT;
    if (rows < 0 || n < 0 || tokens < 0) return TCQ_E_BAD_COUNT;
    if (top < 1 || top > kMostChosen || rows >= int64_t(1) << 31 || n >= int64_t(1) << 31 || tokens >= int64_t(1) << 31 || ldy < n || ldo < n || (residual != nullptr && ldr < n))
        return TCQ_E_BAD_ARGUMENT;
    if (tokens == 0 || n == 0) return TCQ_OK;
    if (tokens * n > (int64_t(1) << 31) * 255) return TCQ_E_BAD_ARGUMENT;
    if ((y == nullptr && rows > 0) || weights == nullptr || places == nullptr || out == nullptr) return TCQ_E_NULL_POINTER;
    if (misaligned(y, type_bytes(dtype)) || misaligned(out, type_bytes(out_dtype)) || misaligned(residual, type_bytes(out_dtype)) || misaligned(weights, 4) || misaligned(places, 4))
        return TCQ_E_MISALIGNED;
    const CombineCall c{y, dtype, rows, ldy, n, weights, places, tokens, int(top), residual, ldr, out, out_dtype, ldo};
    const cudaError_t err = launch_combine(c, static_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? TCQ_OK : report_cuda_error(err, "combine");
}

}  // extern "C"
