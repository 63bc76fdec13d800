// Entry points of the int8 products (int8_gemm.cuh): argument checks and the choice of the kernel.
#include "int8_gemm.cuh"

namespace b200 {

// Sums of K products of magnitude 2^14 at most fit 32 bits up to here.
constexpr int64_t kInt8MaxK = 131071;

static int check_int8(const char* what, const void* a, int64_t lda, const void* b, int64_t ldb, const void* sa, const void* sb,
                      const void* c, int c_dtype, int64_t M, int64_t N, int64_t K) {
  B200_CHECK_ARG(a && b && sa && sb && c, "%s: null pointer", what);
  B200_CHECK_ARG(c_dtype == B200_BF16 || c_dtype == B200_F16 || c_dtype == B200_F32, "%s: unknown dtype code %d", what, c_dtype);
  B200_CHECK_ARG(K > 0, "%s: K is zero", what);
  B200_UNSUPPORTED(K % 16 != 0 || lda % 16 != 0 || ldb % 16 != 0 || (uintptr_t)a % 16 != 0 || (uintptr_t)b % 16 != 0,
                   "%s: rows of 8-bit integers start at multiples of 16 bytes (K=%lld, row strides %lld and %lld)", what, (long long)K,
                   (long long)lda, (long long)ldb);
  B200_CHECK_ARG((M == 1 || lda >= K) && (N == 1 || ldb >= K), "%s: row strides %lld and %lld for K=%lld", what, (long long)lda,
                 (long long)ldb, (long long)K);
  B200_UNSUPPORTED(N % 8 != 0, "%s: N=%lld is not a multiple of 8", what, (long long)N);
  B200_UNSUPPORTED(K > kInt8MaxK, "%s: K=%lld, 32-bit sums hold %lld products", what, (long long)K, (long long)kInt8MaxK);
  B200_UNSUPPORTED(M > 0x7fffff00LL || N > 0x7fffff00LL || cdiv(M, 16) * cdiv(N, 128) > 0x7fffffffLL / 8, "%s: too many tiles", what);
  B200_CHECK_ARG((uintptr_t)c % 16 == 0 && (uintptr_t)sa % 4 == 0 && (uintptr_t)sb % 4 == 0, "%s: misaligned pointer", what);
  return B200_OK;
}

template <typename OutT>
static int run_int8(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t K, Int8Params p, cudaStream_t st) {
  return p.M <= 16 ? launch_int8_stream<16, OutT>(a, lda, b, ldb, K, p, st) : launch_int8_stream<128, OutT>(a, lda, b, ldb, K, p, st);
}

}  // namespace b200

extern "C" int b200_int8_scaled_mm(const void* a, int64_t lda, const float* sa, const void* b, int64_t ldb, const float* sb,
                                   const void* bias, void* c, int c_dtype, int64_t M, int64_t N, int64_t K, void* stream) {
  using namespace b200;
  B200_CHECK_ARG(M >= 0 && N >= 0 && K >= 0, "int8_scaled_mm: negative shape");
  if (M == 0 || N == 0) return B200_OK;
  if (int rc = check_int8("int8_scaled_mm", a, lda, b, ldb, sa, sb, c, c_dtype, M, N, K)) return rc;
  Int8Params p = {};
  p.sa = sa, p.sb = sb, p.bias = bias, p.C = c;
  p.w = static_cast<const int8_t*>(b), p.w_ld = ldb;
  p.M = (int)M, p.N = (int)N, p.num_kb = (int)cdiv(K, kBK);
  p.status = device_status_word();
  if (!p.status) {
    set_error_detail("cannot resolve the device status word");
    return B200_E_LAUNCH;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (c_dtype) {
    case B200_BF16: return run_int8<__nv_bfloat16>(a, lda, b, ldb, K, p, st);
    case B200_F16: return run_int8<__half>(a, lda, b, ldb, K, p, st);
    default: return run_int8<float>(a, lda, b, ldb, K, p, st);
  }
}
