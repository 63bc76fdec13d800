// Entry points of the int8 products (int8_gemm.cuh): argument checks and the choice of the kernel.
#include "int8_gemm.cuh"
#include "int8_gemm_pair.cuh"

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

struct Int8Plan {
  int pair_n;  // columns of a CTA pair's tile; 0: the stream kernel
  int nt, splits;
};

static Int8Plan plan_int8(int64_t M, int64_t N, int64_t K, int sms) {
  Int8Plan pl = {};
  const Tuning& t = tuning();
  const int64_t num_kb = cdiv(K, kBK);
  if (M > 256) pl.pair_n = 256;
  if (t.int8_tile > 0) pl.pair_n = t.int8_tile > 1000 ? (int)t.int8_tile - 1000 : 0;
  if (pl.pair_n) {
    pl.pair_n = pl.pair_n < 32 ? 32 : pl.pair_n > 256 ? 256 : pl.pair_n / 32 * 32;
    pl.splits = t.int8_splits == 2 || t.int8_splits == 4 ? (int)t.int8_splits : 1;
    if (pl.splits > num_kb || cdiv(num_kb, cdiv(num_kb, pl.splits)) != pl.splits) pl.splits = 1;  // no empty split
    return pl;
  }
  const int cap = t.int8_tile > 0 ? (int)t.int8_tile : 256;
  const int64_t t_tiles = cdiv(M, cap);
  pl.nt = (int)align_up(cdiv(M, t_tiles), 16);
  const int64_t items = cdiv(N, 128) * cdiv(M, pl.nt);
  int64_t want = items * 8 <= sms ? 8 : items * 4 <= sms ? 4 : items * 2 <= sms ? 2 : 1;
  if (t.int8_splits > 0) want = t.int8_splits < 8 ? t.int8_splits : 8;
  if (want > num_kb) want = num_kb;
  pl.splits = (int)cdiv(num_kb, cdiv(num_kb, want));  // no empty split
  return pl;
}

template <typename OutT>
static int run_int8(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t K, Int8Params p, cudaStream_t st) {
  const Int8Plan pl = plan_int8(p.M, p.N, K, sm_count());
  p.nt = pl.pair_n ? pl.pair_n : pl.nt, p.k_splits = pl.splits;
  if (pl.pair_n)
    return pl.pair_n > 128 ? launch_int8_pair<256, OutT>(a, lda, b, ldb, K, p, st) : launch_int8_pair<128, OutT>(a, lda, b, ldb, K, p, st);
  return pl.nt <= 16    ? launch_int8_stream<16, OutT>(a, lda, b, ldb, K, p, st)
         : pl.nt <= 32  ? launch_int8_stream<32, OutT>(a, lda, b, ldb, K, p, st)
         : pl.nt <= 64  ? launch_int8_stream<64, OutT>(a, lda, b, ldb, K, p, st)
         : pl.nt <= 128 ? launch_int8_stream<128, OutT>(a, lda, b, ldb, K, p, st)
                        : launch_int8_stream<256, OutT>(a, lda, b, ldb, K, p, st);
}

// Checked operands.
static int run_int8(const void* a, int64_t lda, const float* sa, const void* b, int64_t ldb, const float* sb, const void* bias, void* c,
                    int c_dtype, int64_t M, int64_t N, int64_t K, cudaStream_t st) {
  Int8Params p = {};
  p.sa = sa, p.sb = sb, p.bias = bias, p.C = c;
  p.w = static_cast<const int8_t*>(b), p.w_ld = ldb;
  p.M = (int)M, p.N = (int)N, p.num_kb = (int)cdiv(K, kBK);
  p.status = device_status_word();
  if (!p.status) {
    set_error_detail("cannot resolve the device status word");
    return B200_E_LAUNCH;
  }
  switch (c_dtype) {
    case B200_BF16: return run_int8<__nv_bfloat16>(a, lda, b, ldb, K, p, st);
    case B200_F16: return run_int8<__half>(a, lda, b, ldb, K, p, st);
    default: return run_int8<float>(a, lda, b, ldb, K, p, st);
  }
}

}  // namespace b200

extern "C" int b200_int8_scaled_mm(const void* a, int64_t lda, const float* sa, const void* b, int64_t ldb, const float* sb,
                                   const void* bias, void* c, int c_dtype, int64_t M, int64_t N, int64_t K, void* stream) {
  using namespace b200;
  B200_CHECK_ARG(M >= 0 && N >= 0 && K >= 0, "int8_scaled_mm: negative shape");
  if (M == 0 || N == 0) return B200_OK;
  if (int rc = check_int8("int8_scaled_mm", a, lda, b, ldb, sa, sb, c, c_dtype, M, N, K)) return rc;
  return run_int8(a, lda, sa, b, ldb, sb, bias, c, c_dtype, M, N, K, static_cast<cudaStream_t>(stream));
}

extern "C" size_t b200_w8a8_int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  (void)N;
  return M > 0 && K > 0 ? b200::align_up((size_t)M * K, 16) + (size_t)M * 4 : 0;
}

extern "C" int b200_w8a8_int8_linear(const void* x, int64_t x_ld, int x_dtype, const void* w, int64_t ldw, const float* sw,
                                     const void* bias, void* out, int64_t M, int64_t N, int64_t K, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  using namespace b200;
  B200_CHECK_ARG(M >= 0 && N >= 0 && K >= 0, "w8a8_int8_linear: negative shape");
  if (M == 0 || N == 0) return B200_OK;
  B200_CHECK_ARG(x_dtype == B200_BF16 || x_dtype == B200_F16, "w8a8_int8_linear: input dtype code %d", x_dtype);
  if (workspace == nullptr || workspace_bytes < b200_w8a8_int8_linear_workspace_bytes(M, N, K)) {
    set_error_detail("w8a8_int8_linear: workspace of %zu bytes, %zu needed", workspace_bytes, b200_w8a8_int8_linear_workspace_bytes(M, N, K));
    return B200_E_WORKSPACE;
  }
  void* q = workspace;
  float* s = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + align_up((size_t)M * K, 16));
  if (int rc = check_int8("w8a8_int8_linear", q, K, w, ldw, s, sw, out, x_dtype, M, N, K)) return rc;
  if (int rc = b200_per_token_quant_int8(x, x_ld, x_dtype, q, s, M, K, 0, stream)) return rc;
  return run_int8(q, K, s, w, ldw, sw, bias, out, x_dtype, M, N, K, static_cast<cudaStream_t>(stream));
}
