// ops_linear.cu -- int8 product with a scale for each token and each channel
// (include/czg_ops.h): the row quantiser and the product.
#include <cmath>
#include <string>

#include "ops_common.cuh"

namespace czg {

static thread_local std::string g_ops_error;

int ops_fail(int status, const char *why) {
    g_ops_error = why;
    return status;
}
int ops_cuda(cudaError_t e) {
    if (e == cudaSuccess) return CZG_OK;
    (void)cudaGetLastError();   // a refused launch leaves no error behind for the next caller
    return ops_fail(CZG_E_DEVICE, cudaGetErrorString(e));
}

namespace {

// code = rne(127 x / a).  For 16-bit x the product is exact in fp32 (7 + 11 bits), and the
// rounded quotient falls on a half only where the exact one does: with x = X 2^i, a = A 2^j
// (X, A < 2^11) a quotient q that is no half is 1 / (2 A 2^(j-i)) >= |q| 2^-19 away from
// one, and the division is off by |q| 2^-24 at most.  (fp32 x: both steps round.)
// Rows of values beyond 2^100 are scaled by 2^-20 first, which leaves the quotients alone.
__device__ __forceinline__ int code_of(float x, float a) {
    return (int)rintf(__fdiv_rn(x * 127.0f, a));
}

// One CTA a row: the row's maximum, then its codes.
template <typename T>
__global__ void __launch_bounds__(256) k_quantize_rows(const T *__restrict__ x, int64_t ldx, int64_t k,
                                                       int8_t *__restrict__ codes, int64_t ldc, float *__restrict__ scales) {
    const T *row = x + (int64_t)blockIdx.x * ldx;
    int8_t *out = codes + (int64_t)blockIdx.x * ldc;
    __shared__ float part[8];
    float a = 0.0f;
    bool bad = false;
    for (int64_t i = threadIdx.x; i < k; i += 256) {
        const float v = fabsf(to_f32(row[i]));
        bad |= !(v <= 3.402823466e38f);
        a = fmaxf(a, v);
    }
    if (bad) a = INFINITY;   // NaN and infinities both end as a row of NaN
    for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
    __syncthreads();
    for (int w = 0; w < 8; w++) a = fmaxf(a, part[w]);
    const bool fine = a <= 3.402823466e38f;
    if (threadIdx.x == 0) scales[blockIdx.x] = fine ? __fdiv_rn(a, 127.0f) : NAN;
    const float f = a > 1.2676506e30f ? 9.5367431640625e-7f : 1.0f;
    const int64_t kp = (k + 15) & ~(int64_t)15;
    for (int64_t i = threadIdx.x; i < kp; i += 256)
        out[i] = i < k && fine && a > 0.0f ? (int8_t)code_of(to_f32(row[i]) * f, a * f) : (int8_t)0;
}

// One thread an output, four products an instruction; rows and columns past the ends
// read row 0, whose sum is thrown away.
template <typename T>
__global__ void __launch_bounds__(256) k_linear_i8(const int8_t *__restrict__ x, int64_t ldx, const float *__restrict__ xs,
                                                   const int8_t *__restrict__ w, int64_t ldw, const float *__restrict__ ws,
                                                   const float *__restrict__ bias, int64_t m, int64_t n, int64_t k,
                                                   T *__restrict__ out, int64_t ldo) {
    const int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), j = (int64_t)blockIdx.y * 16 + (threadIdx.x & 15);
    if (i >= m || j >= n) return;
    const int8_t *a = x + i * ldx, *b = w + j * ldw;
    int acc = 0;
    int64_t c = 0;
    for (; c + 4 <= k; c += 4)
        acc = __dp4a(*reinterpret_cast<const int *>(a + c), *reinterpret_cast<const int *>(b + c), acc);
    for (; c < k; c++) acc += (int)a[c] * b[c];
    float y = __fmul_rn(__fmul_rn((float)acc, xs[i]), ws[j]);
    if (bias) y = __fadd_rn(y, bias[j]);
    out[i * ldo + j] = from_f32<T>(y);
}

template <typename T>
int quantize(const void *x, int64_t ldx, int64_t m, int64_t k, int8_t *codes, int64_t ldc, float *scales, cudaStream_t st) {
    k_quantize_rows<T><<<(unsigned)m, 256, 0, st>>>(static_cast<const T *>(x), ldx, k, codes, ldc, scales);
    return ops_cuda(cudaGetLastError());
}

int quantize_any(const void *x, int dtype, int64_t ldx, int64_t m, int64_t k, int8_t *codes, int64_t ldc, float *scales,
                 cudaStream_t st) {
    if (dtype == CZG_F32) return quantize<float>(x, ldx, m, k, codes, ldc, scales, st);
    if (dtype == CZG_BF16) return quantize<__nv_bfloat16>(x, ldx, m, k, codes, ldc, scales, st);
    return quantize<__half>(x, ldx, m, k, codes, ldc, scales, st);
}

template <typename T>
int linear(const int8_t *x, int64_t ldx, const float *xs, const int8_t *w, int64_t ldw, const float *ws, const float *bias,
           int64_t m, int64_t n, int64_t k, void *out, int64_t ldo, cudaStream_t st) {
    const dim3 grid((unsigned)((m + 15) / 16), (unsigned)((n + 15) / 16));
    k_linear_i8<T><<<grid, 256, 0, st>>>(x, ldx, xs, w, ldw, ws, bias, m, n, k, static_cast<T *>(out), ldo);
    return ops_cuda(cudaGetLastError());
}

int linear_any(const int8_t *x, int64_t ldx, const float *xs, const int8_t *w, int64_t ldw, const float *ws,
               const float *bias, int64_t m, int64_t n, int64_t k, void *out, int dtype, int64_t ldo, cudaStream_t st) {
    if (dtype == CZG_F32) return linear<float>(x, ldx, xs, w, ldw, ws, bias, m, n, k, out, ldo, st);
    if (dtype == CZG_BF16) return linear<__nv_bfloat16>(x, ldx, xs, w, ldw, ws, bias, m, n, k, out, ldo, st);
    return linear<__half>(x, ldx, xs, w, ldw, ws, bias, m, n, k, out, ldo, st);
}

const char *check_codes(const int8_t *p, int64_t ld, int64_t rows, int64_t k) {
    if (!aligned(p, 16) || ld % 16 != 0) return "rows of codes must begin on 16-byte boundaries";
    if (rows > 1 && ld < k) return "rows of codes overlap";
    return nullptr;
}

int check_linear(const int8_t *w, int64_t ldw, const float *ws, int64_t m, int64_t n, int64_t k, const void *out,
                 int out_dtype, int64_t ldo) {
    if (!w || !ws || !out) return ops_fail(CZG_E_ARG, "null pointer");
    if (!dtype_ok(out_dtype)) return ops_fail(CZG_E_ARG, "unknown out_dtype");
    if (const char *why = check_codes(w, ldw, n, k)) return ops_fail(CZG_E_ARG, why);
    if (!aligned(out, (uintptr_t)elem_bytes(out_dtype))) return ops_fail(CZG_E_ARG, "out is not aligned to its type");
    if (m > 1 && ldo < n) return ops_fail(CZG_E_ARG, "rows of out overlap");
    return CZG_OK;
}

int check_sizes(int64_t m, int64_t n, int64_t k) {
    if (m < 0 || n < 0 || k < 1) return ops_fail(CZG_E_ARG, "m and n must not be negative, k must be at least 1");
    if (k > CZG_LINEAR_MAX_K) return ops_fail(CZG_E_LIMIT, "k is beyond CZG_LINEAR_MAX_K");
    if (m > 0x7FFFFFFF || n > 0x7FFFFFFF) return ops_fail(CZG_E_LIMIT, "m and n must be below 2^31");
    return CZG_OK;
}

int check_x(const void *x, int dtype, int64_t ldx, int64_t m, int64_t k) {
    if (!x) return ops_fail(CZG_E_ARG, "null pointer");
    if (!dtype_ok(dtype)) return ops_fail(CZG_E_ARG, "unknown dtype");
    if (!aligned(x, (uintptr_t)elem_bytes(dtype))) return ops_fail(CZG_E_ARG, "x is not aligned to its type");
    if (m > 1 && ldx < 0) return ops_fail(CZG_E_ARG, "ld_x is negative");
    return CZG_OK;
}

int64_t codes_ld(int64_t k) { return (k + 15) & ~(int64_t)15; }

}  // namespace
}  // namespace czg

using namespace czg;

extern "C" const char *czg_ops_last_error(void) { return g_ops_error.c_str(); }

extern "C" int czg_quantize_rows(const void *x, int dtype, int64_t ld_x, int64_t m, int64_t k, int8_t *codes,
                                 int64_t ld_codes, float *scales, void *stream) {
    if (m < 0 || k < 1) return ops_fail(CZG_E_ARG, "m must not be negative, k must be at least 1");
    if (m > 0x7FFFFFFF) return ops_fail(CZG_E_LIMIT, "m must be below 2^31");
    if (m == 0) return CZG_OK;
    if (int st = check_x(x, dtype, ld_x, m, k)) return st;
    if (!codes || !scales) return ops_fail(CZG_E_ARG, "null pointer");
    if (const char *why = check_codes(codes, ld_codes, m, codes_ld(k))) return ops_fail(CZG_E_ARG, why);
    return quantize_any(x, dtype, ld_x, m, k, codes, ld_codes, scales, static_cast<cudaStream_t>(stream));
}

extern "C" int czg_linear_i8(const int8_t *x, int64_t ld_x, const float *x_scale, const int8_t *w, int64_t ld_w,
                             const float *w_scale, const float *bias, int64_t m, int64_t n, int64_t k, void *out,
                             int out_dtype, int64_t ld_out, void *stream) {
    if (int st = check_sizes(m, n, k)) return st;
    if (m == 0 || n == 0) return CZG_OK;
    if (!x || !x_scale) return ops_fail(CZG_E_ARG, "null pointer");
    if (const char *why = check_codes(x, ld_x, m, k)) return ops_fail(CZG_E_ARG, why);
    if (int st = check_linear(w, ld_w, w_scale, m, n, k, out, out_dtype, ld_out)) return st;
    return linear_any(x, ld_x, x_scale, w, ld_w, w_scale, bias, m, n, k, out, out_dtype, ld_out,
                      static_cast<cudaStream_t>(stream));
}

extern "C" uint64_t czg_linear_i8_workspace(int64_t m, int64_t k) {
    if (m <= 0 || k <= 0) return 0;
    return (uint64_t)m * (uint64_t)codes_ld(k) + (((uint64_t)m * 4 + 15) & ~15ull);
}

extern "C" int czg_linear_i8_dynamic(const void *x, int dtype, int64_t ld_x, const int8_t *w, int64_t ld_w,
                                     const float *w_scale, const float *bias, int64_t m, int64_t n, int64_t k,
                                     void *out, int out_dtype, int64_t ld_out, void *ws, uint64_t ws_bytes, void *stream) {
    if (int st = check_sizes(m, n, k)) return st;
    if (m == 0 || n == 0) return CZG_OK;
    if (int st = check_x(x, dtype, ld_x, m, k)) return st;
    if (int st = check_linear(w, ld_w, w_scale, m, n, k, out, out_dtype, ld_out)) return st;
    if (!ws || !aligned(ws, 16)) return ops_fail(CZG_E_ARG, "the workspace must begin on a 16-byte boundary");
    if (ws_bytes < czg_linear_i8_workspace(m, k)) return ops_fail(CZG_E_ARG, "the workspace is too small");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int8_t *codes = static_cast<int8_t *>(ws);
    float *scales = reinterpret_cast<float *>(codes + m * codes_ld(k));
    if (int e = quantize_any(x, dtype, ld_x, m, k, codes, codes_ld(k), scales, st)) return e;
    return linear_any(codes, codes_ld(k), scales, w, ld_w, w_scale, bias, m, n, k, out, out_dtype, ld_out, st);
}
