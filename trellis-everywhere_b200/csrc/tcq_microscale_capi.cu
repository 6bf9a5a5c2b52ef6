// C ABI of the 4-bit microscaled operators (declared in include/tcq_b200.h): argument checks.
#include "../../include/tcq_b200.h"

#include "tcq_microscale.cuh"

using namespace tcq;

namespace {

bool misaligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }
constexpr int64_t kMostRows = int64_t(1) << 31;          // grids and coordinates fit 32 bits
constexpr int64_t kMostColumns = int64_t(1) << 24;       // a tile's products end well within the limit of a wait for them

int check_ms(int64_t rows, int64_t k, int format, int dtype) {
    if (format != TCQ_MS_MXFP4 && format != TCQ_MS_NVFP4) return TCQ_E_BAD_FORMAT;
    if (dtype < TCQ_F32 || dtype > TCQ_BF16) return TCQ_E_BAD_FORMAT;
    if (rows < 0 || k < 0) return TCQ_E_BAD_COUNT;
    return rows >= kMostRows || k > kMostColumns ? TCQ_E_BAD_ARGUMENT : TCQ_OK;
}
// One matrix in 4 bits: what must be there, and aligned.
int check_ms_matrix(const void* codes, const void* scales, const void* row_scale, int format) {
    if (!codes || !scales || (format == TCQ_MS_NVFP4) != (row_scale != nullptr)) return TCQ_E_NULL_POINTER;
    return misaligned(codes, 16) || misaligned(scales, 16) || misaligned(row_scale, 4) ? TCQ_E_MISALIGNED : TCQ_OK;
}
size_t type_bytes(int dtype) { return dtype == TCQ_F32 ? 4 : 2; }

int linear_core(const void* x, int dtype, int64_t m, int64_t ldx, const uint8_t* codes, const uint8_t* scales, const float* row_scale, int64_t n, int64_t k,
                int format, void* y, int64_t ldy, void* ws, size_t ws_bytes, unsigned loads, void* stream) {
    int rc = check_ms(n, k, format, dtype);
    if (rc == TCQ_OK) rc = check_ms(m, k, format, dtype);
    if (rc != TCQ_OK) return rc;
    if (n == 0 || m == 0) return TCQ_OK;
    if (k == 0 || ldx < k || ldy < n) return TCQ_E_BAD_ARGUMENT;
    const bool direct = ms_linear_direct(x, dtype, m, ldx, format);
    if (x == nullptr || y == nullptr || (ws == nullptr && !direct)) return TCQ_E_NULL_POINTER;
    if ((rc = check_ms_matrix(codes, scales, row_scale, format)) != TCQ_OK) return rc;
    if (misaligned(x, type_bytes(dtype)) || misaligned(y, type_bytes(dtype)) || misaligned(ws, 256)) return TCQ_E_MISALIGNED;
    if (!direct && ws_bytes < ms_linear_workspace_bytes(m, n, k, dtype, format)) return TCQ_E_WORKSPACE;
    cudaError_t err = launch_ms_linear(x, dtype, m, ldx, {codes, scales, row_scale, n}, k, format, y, ldy, ws, loads, static_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? TCQ_OK : report_cuda_error(err, "ms_linear");
}

int matmul_core(const uint8_t* x_codes, const uint8_t* x_scales, const float* x_row_scale, int64_t m, const uint8_t* codes, const uint8_t* scales,
                const float* row_scale, int64_t n, int64_t k, int format, void* y, int dtype, int64_t ldy, unsigned loads, void* stream) {
    int rc = check_ms(n, k, format, dtype);
    if (rc == TCQ_OK) rc = check_ms(m, k, format, dtype);
    if (rc != TCQ_OK) return rc;
    if (n == 0 || m == 0) return TCQ_OK;
    if (k == 0 || ldy < n) return TCQ_E_BAD_ARGUMENT;
    if (y == nullptr) return TCQ_E_NULL_POINTER;
    if ((rc = check_ms_matrix(x_codes, x_scales, x_row_scale, format)) != TCQ_OK) return rc;
    if ((rc = check_ms_matrix(codes, scales, row_scale, format)) != TCQ_OK) return rc;
    if (misaligned(y, type_bytes(dtype))) return TCQ_E_MISALIGNED;
    cudaError_t err = launch_ms_matmul({x_codes, x_scales, x_row_scale, m}, {codes, scales, row_scale, n}, k, format, y, dtype, ldy, loads,
                                       static_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? TCQ_OK : report_cuda_error(err, "ms_matmul");
}
bool bad_loads(int64_t loads) { return loads < 0 || loads >= int64_t(kMsAllLoads); }

}  // namespace

extern "C" {

size_t tcq_ms_code_pitch(int64_t k) { return k < 0 ? 0 : size_t(ms_pitch(k)); }

size_t tcq_ms_scale_bytes(int64_t rows, int64_t k, int format) {
    return check_ms(rows, k, format, TCQ_F32) != TCQ_OK ? 0 : size_t(ms_scale_bytes(rows, k, format));
}

int tcq_ms_quantize(const void* x, int dtype, int64_t rows, int64_t k, int64_t ldx, int format, int rotate, const float* signs,
                    uint8_t* codes, uint8_t* scales, float* row_scale, void* stream) {
    int rc = check_ms(rows, k, format, dtype);
    if (rc != TCQ_OK) return rc;
    if (rotate != 0 && rotate != 16 && rotate != 32 && rotate != 64 && rotate != 128) return TCQ_E_BAD_ARGUMENT;
    if (rotate != 0 && k % rotate) return TCQ_E_BAD_ARGUMENT;
    if (rows == 0 || k == 0) return TCQ_OK;
    if (ldx < k) return TCQ_E_BAD_ARGUMENT;
    if (x == nullptr || (rotate != 0) != (signs != nullptr)) return TCQ_E_NULL_POINTER;
    if ((rc = check_ms_matrix(codes, scales, row_scale, format)) != TCQ_OK) return rc;
    if (misaligned(x, type_bytes(dtype)) || misaligned(signs, 4)) return TCQ_E_MISALIGNED;
    cudaError_t err = launch_ms_quantize(x, dtype, rows, k, ldx, format, rotate, signs, codes, scales, row_scale,
                                         static_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? TCQ_OK : report_cuda_error(err, "ms_quantize");
}

int tcq_ms_dequantize(const uint8_t* codes, const uint8_t* scales, const float* row_scale, int64_t rows, int64_t k, int format,
                      void* out, int dtype, int64_t ldo, void* stream) {
    int rc = check_ms(rows, k, format, dtype);
    if (rc != TCQ_OK) return rc;
    if (rows == 0 || k == 0) return TCQ_OK;
    if (ldo < k) return TCQ_E_BAD_ARGUMENT;
    if (out == nullptr) return TCQ_E_NULL_POINTER;
    if ((rc = check_ms_matrix(codes, scales, row_scale, format)) != TCQ_OK) return rc;
    if (misaligned(out, type_bytes(dtype))) return TCQ_E_MISALIGNED;
    cudaError_t err = launch_ms_dequantize({codes, scales, row_scale, rows}, k, format, out, dtype, ldo, static_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? TCQ_OK : report_cuda_error(err, "ms_dequantize");
}

size_t tcq_ms_linear_workspace_bytes(int64_t m, int64_t n, int64_t k, int dtype, int format) {
    return check_ms(m, k, format, dtype) != TCQ_OK || check_ms(n, k, format, dtype) != TCQ_OK ? 0 : ms_linear_workspace_bytes(m, n, k, dtype, format);
}

int tcq_ms_linear(const void* x, int dtype, int64_t m, int64_t ldx, const uint8_t* codes, const uint8_t* scales,
                  const float* row_scale, int64_t n, int64_t k, int format, void* y, int64_t ldy, void* ws, size_t ws_bytes,
                  void* stream) {
    return linear_core(x, dtype, m, ldx, codes, scales, row_scale, n, k, format, y, ldy, ws, ws_bytes, kMsAllLoads, stream);
}

int tcq_ms_matmul(const uint8_t* x_codes, const uint8_t* x_scales, const float* x_row_scale, int64_t m, const uint8_t* codes,
                  const uint8_t* scales, const float* row_scale, int64_t n, int64_t k, int format, void* y, int dtype,
                  int64_t ldy, void* stream) {
    return matmul_core(x_codes, x_scales, x_row_scale, m, codes, scales, row_scale, n, k, format, y, dtype, ldy, kMsAllLoads, stream);
}

int tcq_selftest_ms_linear_waits(int64_t loads, const void* x, int dtype, int64_t m, int64_t ldx, const uint8_t* codes, const uint8_t* scales,
                                 const float* row_scale, int64_t n, int64_t k, int format, void* y, int64_t ldy, void* ws, size_t ws_bytes,
                                 void* stream) {
    return bad_loads(loads) ? TCQ_E_BAD_COUNT
                            : linear_core(x, dtype, m, ldx, codes, scales, row_scale, n, k, format, y, ldy, ws, ws_bytes, unsigned(loads), stream);
}

int tcq_selftest_ms_matmul_waits(int64_t loads, const uint8_t* x_codes, const uint8_t* x_scales, const float* x_row_scale, int64_t m,
                                 const uint8_t* codes, const uint8_t* scales, const float* row_scale, int64_t n, int64_t k, int format,
                                 void* y, int dtype, int64_t ldy, void* stream) {
    return bad_loads(loads) ? TCQ_E_BAD_COUNT
                            : matmul_core(x_codes, x_scales, x_row_scale, m, codes, scales, row_scale, n, k, format, y, dtype, ldy, unsigned(loads), stream);
}

}  // extern "C"
