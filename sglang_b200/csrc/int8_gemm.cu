// Entry points of the int8 products (int8_gemm.cuh): argument checks and the choice of the kernel.
#include <math.h>

#include "int8_gemm.cuh"
#include "int8_gemm_pair.cuh"

namespace b200 {

// Sums of K products of magnitude 2^14 at most fit 32 bits up to here.
constexpr int64_t kInt8MaxK = 131071;

static int check_int8(const char* what, const void* a, int64_t lda, const void* b, int64_t ldb, const void* sa, const void* sb,
                      const void* bias, const void* c, int c_dtype, int64_t M, int64_t N, int64_t K) {
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
  B200_CHECK_ARG((uintptr_t)c % 16 == 0 && (uintptr_t)sa % 4 == 0 && (uintptr_t)sb % 4 == 0 &&
                     (uintptr_t)bias % (c_dtype == B200_F32 ? 4 : 2) == 0,
                 "%s: misaligned pointer", what);
  return B200_OK;
}

enum Int8Kernel { INT8_STREAM = 0, INT8_PAIR = 1, INT8_PAIR_SWAPPED = 2 };

struct Int8Plan {
  int kernel;
  int tile, splits;  // tile: tokens (stream, swapped pair) or channels (pair)
  float us;    // what the model expects
};

// Clusters of 1 .. 8 CTAs that a chip of 148 SMs holds at one CTA per SM (as the occupancy query of the runtime says); GPCs are not all
// of the same size, so large clusters leave SMs empty.
static int clusters_at_once(int size, int sms) {
  static const int on_148[9] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
  const int n = on_148[size] * sms / 148;
  return n > 0 ? n : 1;
}

static float join(float a, float b) {  // near the larger of the two, a little above where they are alike
  a *= a, b *= b;
  return sqrtf(sqrtf(a * a + b * b));
}

// Time of one call in us, back to back with others: started from a least-squares fit, the constants were then moved until the choice
// among 10468 measured sizes (1 to 4096 rows, N 256 to 57344, K 256 to 28672, each with every tile and split below) was as near the
// best of them as it would come. The sizes of the served models and their shards, half of them all, weigh three times as much as the others, and what is
// more than 5 % behind counts double. Behind the best on 5521 other sizes: 0.5 % on average up to 16 rows, 0.6 to 1.9 % above; 2 and 6 %
// at the 90th percentile, 6 and 8 to 21 % at the 99th; at worst 18 %, and 54 % between 33 and 64 rows.
struct StreamCost {
  float start, alone, alone_nt, shared, shared_nt;  // a K block of a CTA that has its SM to itself, of one of several on an SM
  float bandwidth, store_nt, sum, sum_nt, cta, wave;
};
static float stream_us(int64_t M, int64_t N, int64_t K, int nt, int splits, int sms) {
  static const StreamCost few = {1.34f, 0.2743f, 0.0026f, 0.1973f, 0.f, 5.91e6f, 0.0034f, 0.435f, 0.f, 0.682f, 0.63f};
  static const StreamCost some = {2.28f, 0.2091f, 0.0017f, 0.1168f, 0.0016f, 10.62e6f, 0.0148f, 0.482f, 0.0127f, 0.770f, 0.42f};
  static const StreamCost many = {1.97f, 0.2161f, 0.0010f, 0.1137f, 0.0022f, 9.43e6f, 0.0109f, 0.350f, 0.0177f, 0.722f, 0.73f};
  const StreamCost& c = M <= 16 ? few : M <= 64 ? some : many;
  const int per_sm = nt <= 64 ? 2 : 1;
  const int64_t items = cdiv(N, 128) * cdiv(M, nt), kbs = cdiv(cdiv(K, kBK), splits);
  const int64_t per = cdiv(items, clusters_at_once(splits, sms)), waves = cdiv(per, per_sm);
  const float alone = c.alone + c.alone_nt * nt, shared = c.shared + c.shared_nt * nt;
  const float rate = per <= 1 || per_sm == 1 ? alone : alone / 2 > shared ? alone / 2 : shared;
  const float memory = ((float)N * K + (float)M * K + 2.f * M * N) / c.bandwidth;
  const float sum = splits > 1 ? c.sum + c.sum_nt * nt * (splits - 1) / splits : 0.f;
  return c.start + join(per * kbs * rate, memory) + (c.store_nt * nt + sum) * waves + c.cta * items * splits / sms + c.wave * (waves - 1);
}
static float pair_us(int64_t M, int64_t N, int64_t K, bool swap, int bn, int splits, int sms) {
  const int64_t tiles = swap ? cdiv(M, bn) * cdiv(N, 2 * kBM) : cdiv(N, bn) * cdiv(M, 2 * kBM), kbs = cdiv(cdiv(K, kBK), splits);
  const int64_t waves = cdiv(tiles, clusters_at_once(2 * splits, sms));
  const float loop = kbs * (0.1221f + 0.0009f * bn), epilogue = 1.04f + (swap ? 0.0088f : 0.0074f) * bn;
  const float memory = ((float)N * K + (float)M * K + 2.f * M * N) / 8.27e6f;
  const float sum = splits > 1 ? 1.15f + 0.0197f * bn * (splits - 1) / splits : 0.f;
  return (swap ? 3.57f : 3.47f) + join((waves - 1) * (loop > epilogue ? loop : epilogue) + loop, memory) + (swap ? 0.0040f : 0.0036f) * bn + sum * waves;
}

static Int8Plan plan_int8(int64_t M, int64_t N, int64_t K, int sms) {
  const Tuning& t = tuning();
  const int64_t num_kb = cdiv(K, kBK);
  const int forced = t.int8_splits > 0 ? (int)t.int8_splits : 0;
  // no split without a K block
  auto whole = [&](int splits) { return splits <= num_kb && cdiv(num_kb, cdiv(num_kb, splits)) == splits; };
  Int8Plan best = {INT8_STREAM, 16, 1, 1e30f};
  auto consider = [&](int kernel, int tile, int splits) {
    if (!whole(splits)) return;
    const float us = kernel == INT8_STREAM ? stream_us(M, N, K, tile, splits, sms)
                                           : pair_us(M, N, K, kernel == INT8_PAIR_SWAPPED, tile, splits, sms);
    if (us < best.us) best = {kernel, tile, splits, us};
  };
  if (t.int8_tile > 1000) {
    const int bn = (int)(t.int8_tile % 1000) / 32 * 32;
    consider(t.int8_tile > 2000 ? INT8_PAIR_SWAPPED : INT8_PAIR, bn < 32 ? 32 : bn > 256 ? 256 : bn,
             (forced == 2 || forced == 4) && whole(forced) ? forced : 1);
    return best;
  }
  if (t.int8_tile > 0) {
    const int cap = t.int8_tile < 16 ? 16 : t.int8_tile > 256 ? 256 : (int)t.int8_tile / 16 * 16;
    int splits = forced > kInt8MaxSplits ? kInt8MaxSplits : forced > 0 ? forced : 1;
    while (!whole(splits)) --splits;
    consider(INT8_STREAM, (int)align_up(cdiv(M, cdiv(M, cap)), 16), splits);
    return best;
  }
  // the tokens in up to eight tiles of equal size
  for (int64_t tiles = cdiv(M, 256), last = 0; tiles <= 8; ++tiles) {
    const int64_t nt = align_up(cdiv(M, tiles), 16);
    if (nt == last) continue;
    last = nt;
    for (int splits = 1; splits <= kInt8MaxSplits; ++splits)
      if (splits == 1 || cdiv(N, 128) * cdiv(M, nt) * splits <= 2 * sms) consider(INT8_STREAM, (int)nt, splits);
    if (nt == 16) break;
  }
  if (M > 32)
    for (int bn = 32; bn <= 256; bn += 32)
      for (int splits = 1; splits <= 4; splits *= 2) {
        if (splits == 1 || cdiv(N, bn) * cdiv(M, 2 * kBM) * splits <= sms / 2) consider(INT8_PAIR, bn, splits);
        if (bn > 32 && (splits == 1 || cdiv(M, bn) * cdiv(N, 2 * kBM) * splits <= sms / 2)) consider(INT8_PAIR_SWAPPED, bn, splits);
      }
  return best;
}

template <typename OutT>
static int run_int8(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t K, Int8Params p, cudaStream_t st) {
  const Int8Plan pl = plan_int8(p.M, p.N, K, sm_count());
  p.nt = pl.tile, p.k_splits = pl.splits;
  if (pl.kernel == INT8_PAIR)
    return pl.tile > 128 ? launch_int8_pair<256, false, OutT>(a, lda, b, ldb, K, p, st)
                         : launch_int8_pair<128, false, OutT>(a, lda, b, ldb, K, p, st);
  if (pl.kernel == INT8_PAIR_SWAPPED)
    return pl.tile > 128 ? launch_int8_pair<256, true, OutT>(a, lda, b, ldb, K, p, st)
                         : launch_int8_pair<128, true, OutT>(a, lda, b, ldb, K, p, st);
  return pl.tile <= 16    ? launch_int8_stream<16, false, OutT>(a, lda, b, ldb, K, p, st)
         : pl.tile <= 32  ? launch_int8_stream<32, false, OutT>(a, lda, b, ldb, K, p, st)
         : pl.tile <= 64  ? launch_int8_stream<64, false, OutT>(a, lda, b, ldb, K, p, st)
         : pl.tile <= 128 ? launch_int8_stream<128, false, OutT>(a, lda, b, ldb, K, p, st)
                        : launch_int8_stream<256, false, OutT>(a, lda, b, ldb, K, p, st);
}

static int fill_int8(Int8Params& p, const float* sa, const void* b, int64_t ldb, const float* sb, const void* bias, void* c, int64_t M,
                     int64_t N, int64_t K) {
  p = {};
  p.sa = sa, p.sb = sb, p.bias = bias, p.C = c;
  p.w = static_cast<const int8_t*>(b), p.w_ld = ldb;
  p.M = (int)M, p.N = (int)N, p.num_kb = (int)cdiv(K, kBK);
  p.status = device_status_word();
  if (p.status) return B200_OK;
  set_error_detail("cannot resolve the device status word");
  return B200_E_LAUNCH;
}

// Checked operands.
static int run_int8(const void* a, int64_t lda, const float* sa, const void* b, int64_t ldb, const float* sb, const void* bias, void* c,
                    int c_dtype, int64_t M, int64_t N, int64_t K, cudaStream_t st) {
  Int8Params p;
  if (int rc = fill_int8(p, sa, b, ldb, sb, bias, c, M, N, K)) return rc;
  switch (c_dtype) {
    case B200_BF16: return run_int8<__nv_bfloat16>(a, lda, b, ldb, K, p, st);
    case B200_F16: return run_int8<__half>(a, lda, b, ldb, K, p, st);
    default: return run_int8<float>(a, lda, b, ldb, K, p, st);
  }
}

}  // namespace b200

extern "C" int b200_plan_int8(int64_t M, int64_t N, int64_t K, int sms, int* kernel, int* tile, int* splits) {
  using namespace b200;
  B200_CHECK_ARG(M > 0 && N > 0 && K > 0 && sms >= 0 && kernel && tile && splits, "plan_int8: empty shape or null pointer");
  const Int8Plan pl = plan_int8(M, N, K, sms > 0 ? sms : sm_count());
  *kernel = pl.kernel, *tile = pl.tile, *splits = pl.splits;
  return B200_OK;
}

extern "C" int b200_int8_scaled_mm(const void* a, int64_t lda, const float* sa, const void* b, int64_t ldb, const float* sb,
                                   const void* bias, void* c, int c_dtype, int64_t M, int64_t N, int64_t K, void* stream) {
  using namespace b200;
  B200_CHECK_ARG(M >= 0 && N >= 0 && K >= 0, "int8_scaled_mm: negative shape");
  if (M == 0 || N == 0) return B200_OK;
  if (int rc = check_int8("int8_scaled_mm", a, lda, b, ldb, sa, sb, bias, c, c_dtype, M, N, K)) return rc;
  return run_int8(a, lda, sa, b, ldb, sb, bias, c, c_dtype, M, N, K, static_cast<cudaStream_t>(stream));
}

namespace b200 {

// One launch for the layer, where the rows are few and short enough that every CTA may look for their largest magnitudes itself, and
// start at multiples of 16 bytes. Two launches and one, replayed from a graph: 1 x 6144 x 4096 8.5, 6.9 us, 1 x 28672 x 4096 23.1, 21.7,
// 1 x 4096 x 14336 13.5, 13.5, 4 x 6144 x 4096 8.4, 8.0; past the limit 4 x 4096 x 6144 8.1, 9.3, 2 x 4096 x 14336 13.7, 14.3; launched from
// Python 7.0, 5.2 us of host time.
static bool linear_fuses(int64_t M, int64_t K, int aligned) {
  if (!aligned || M > Int8StreamCfg<16, true>::kQuantRows || tuning().int8_linear_fused == 0) return false;
  return tuning().int8_linear_fused > 0 || M * K <= 16384;
}

template <typename T>
static int run_int8_linear_fused(const void* x, int64_t x_ld, const void* w, int64_t ldw, int64_t K, Int8Params p, cudaStream_t st) {
  const Int8Plan pl = plan_int8(p.M, p.N, K, sm_count());  // 16 tokens: the stream kernel
  p.x = x, p.x_ld = x_ld;
  p.nt = 16, p.k_splits = pl.kernel == INT8_STREAM ? pl.splits : 1;
  return launch_int8_stream<16, true, T>(nullptr, 0, w, ldw, K, p, st);
}

}  // namespace b200

extern "C" size_t b200_w8a8_int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int x_aligned) {
  (void)N;
  if (M <= 0 || K <= 0 || b200::linear_fuses(M, K, x_aligned)) return 0;
  return b200::align_up((size_t)M * K, 16) + (size_t)M * 4;
}

extern "C" int b200_w8a8_int8_linear(const void* x, int64_t x_ld, int x_dtype, const void* w, int64_t ldw, const float* sw,
                                     const void* bias, void* out, int64_t M, int64_t N, int64_t K, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  using namespace b200;
  B200_CHECK_ARG(M >= 0 && N >= 0 && K >= 0, "w8a8_int8_linear: negative shape");
  if (M == 0 || N == 0) return B200_OK;
  B200_CHECK_ARG(x && (uintptr_t)x % 2 == 0, "w8a8_int8_linear: null or misaligned input");
  B200_CHECK_ARG(x_dtype == B200_BF16 || x_dtype == B200_F16, "w8a8_int8_linear: input dtype code %d", x_dtype);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int aligned = (uintptr_t)x % 16 == 0 && (M == 1 || x_ld % 8 == 0);
  if (linear_fuses(M, K, aligned)) {
    if (int rc = check_int8("w8a8_int8_linear", w, ldw, w, ldw, sw, sw, bias, out, x_dtype, M, N, K)) return rc;
    Int8Params p;
    if (int rc = fill_int8(p, nullptr, w, ldw, sw, bias, out, M, N, K)) return rc;
    return x_dtype == B200_BF16 ? run_int8_linear_fused<__nv_bfloat16>(x, x_ld, w, ldw, K, p, st)
                                : run_int8_linear_fused<__half>(x, x_ld, w, ldw, K, p, st);
  }
  const size_t need = b200_w8a8_int8_linear_workspace_bytes(M, N, K, 0);
  if (workspace == nullptr || workspace_bytes < need || (uintptr_t)workspace % 16 != 0) {
    set_error_detail("w8a8_int8_linear: workspace of %zu bytes, %zu needed, 16-byte aligned", workspace_bytes, need);
    return B200_E_WORKSPACE;
  }
  void* q = workspace;
  float* s = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + align_up((size_t)M * K, 16));
  if (int rc = check_int8("w8a8_int8_linear", q, K, w, ldw, s, sw, bias, out, x_dtype, M, N, K)) return rc;
  if (int rc = b200_per_token_quant_int8(x, x_ld, x_dtype, q, s, M, K, 0, stream)) return rc;
  return run_int8(q, K, s, w, ldw, sw, bias, out, x_dtype, M, N, K, st);
}
