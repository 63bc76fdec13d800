// Rows of 16-bit (or fp32) activations -> 8-bit rows with scales, with what precedes the quantiser in a decoder layer fused in:
//   rmsnorm_quant          h = x (+ r);  y = h * w * rsqrt(mean(h^2) + eps);  r_out = h rounded once
//   per_token_quant_int8   y = x, or silu(gate) * up of rows [gate | up]
// and three ways to hold y in 8 bits:
//   int8      s = max|y| / 127 per row,               q = rint(y / s)
//   fp8       s = max|y| / 448 per 128 columns,       q = e4m3(y / s), fp32 scales with any strides
//   fp8 ue8m0 s = 2^ceil(log2(max|y| / 448)) likewise, exponent bytes packed four groups per int32 word, rows contiguous
// Sums and maxima are fp32; the floor of a maximum is 1e-10 as in the group quantiser. A row or group with a NaN in it gets a NaN
// (int8: as its scale, there is no NaN code; fp8: as codes).
#include "common.cuh"

namespace b200 {

enum RowSource { ROW_PLAIN = 0, ROW_SILU = 1, ROW_NORM = 2, ROW_ADD_NORM = 3 };

struct RowParams {
  const void* x;
  int64_t x_ld;  // elements between rows
  const void* r;
  int64_t r_ld;
  const void* w;
  void* r_out;  // [M, H], contiguous
  uint8_t* q;   // [M, H], contiguous
  void* s;
  int64_t s_sm, s_sg;  // fp8: element strides of the scales; ue8m0: s_sg = words between groups of four
  int64_t rows;
  int H;
  float eps;
};

// max that keeps a NaN: a row must not hide one behind its other values
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// (sum, max) over the block; every thread gets both. red: 64 floats of shared memory, free again after the next barrier.
__device__ __forceinline__ void block_sum_max(float& sum, float& top, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warps == 1) return;
  if (lane == 0) red[warp] = sum, red[32 + warp] = top;
  __syncthreads();
  sum = lane < warps ? red[lane] : 0.f;
  top = lane < warps ? red[32 + lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
}

__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// The nearest whole number of |v| < 2^22, ties to even, in the low bits of the result: adding 1.5 * 2^23 leaves no room for a fraction.
__device__ __forceinline__ uint32_t rint_bits(float v) { return __float_as_uint(v + 12582912.f); }

// x / s rounded to the nearest float, r = 1 / s rounded: one residual step (Markstein)
__device__ __forceinline__ float div_by(float x, float s, float r) {
  const float q = x * r;
  return fmaf(fmaf(-q, s, x), r, q);
}

struct Ue8m0 {
  uint32_t byte;
  float inv;  // 1 / scale
};
__device__ __forceinline__ Ue8m0 ue8m0_of(float amax) {  // the group quantiser's arithmetic
  const uint32_t bits = __float_as_uint(amax * (1.0f / 448.0f));
  Ue8m0 e;
  e.byte = ((bits >> 23) & 0xffu) + ((bits & 0x7fffffu) != 0 ? 1u : 0u);
  e.inv = __uint_as_float((254u - e.byte) << 23);
  return e;
}

template <int KIND>
__device__ __forceinline__ void put_group_scale(const RowParams& p, int64_t row, int g, float scale, uint32_t byte) {
  if constexpr (KIND == B200_ROW_FP8) {
    static_cast<float*>(p.s)[row * p.s_sm + g * p.s_sg] = scale;
  } else {
    uint8_t* dst = static_cast<uint8_t*>(p.s) + ((int64_t)(g >> 2) * p.s_sg + row) * 4 + (g & 3);
    *dst = (uint8_t)byte;
    if ((g + 1) * 128 == p.H)  // bytes of the last word that belong to no group read as zero
      for (int k = (g & 3) + 1; k < 4; ++k) dst[k - (g & 3)] = 0;
  }
}

// A row per block, one element per thread and step, read twice: any width and alignment.
template <typename T, int SRC, int KIND>
__global__ void __launch_bounds__(256) row_quant_any_kernel(const RowParams p) {
  __shared__ float red[64];
  grid_dependency_wait();
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  const T* r = static_cast<const T*>(p.r) + row * p.r_ld;
  const T* w = static_cast<const T*>(p.w);
  const int H = p.H;
  auto value = [&](int i) {
    const float v = to_f32<T>(x[i]);
    if constexpr (SRC == ROW_SILU) return silu_mul(v, to_f32<T>(x[H + i]));
    if constexpr (SRC == ROW_ADD_NORM) return v + to_f32<T>(r[i]);
    return v;
  };
  auto weight = [&](int i) { return SRC >= ROW_NORM ? to_f32<T>(w[i]) : 1.f; };
  float sum = 0.f, top = 0.f;
  for (int i = threadIdx.x; i < H; i += 256) {
    const float h = value(i);
    sum = fmaf(h, h, sum);
    if constexpr (KIND == B200_ROW_INT8) top = max_nan(top, fabsf(h * weight(i)));
    if constexpr (SRC == ROW_ADD_NORM) static_cast<T*>(p.r_out)[row * H + i] = from_f32<T>(h);
  }
  block_sum_max(sum, top, red);
  const float rstd = SRC >= ROW_NORM ? rsqrtf(sum / (float)H + p.eps) : 1.f;
  if constexpr (KIND == B200_ROW_INT8) {
    const float s = __fdiv_rn(max_nan(top * rstd, 1e-10f), 127.f), inv = __frcp_rn(s);
    if (threadIdx.x == 0) static_cast<float*>(p.s)[row] = s;
    for (int i = threadIdx.x; i < H; i += 256)
      p.q[row * H + i] = (uint8_t)rint_bits(div_by(value(i) * weight(i) * rstd, s, inv));
  } else {  // 128 columns: four per lane of a warp
    for (int g = threadIdx.x >> 5; g * 128 < H; g += 8) {
      const int i0 = g * 128 + (threadIdx.x & 31) * 4;
      float y[4], amax = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        y[k] = value(i0 + k) * weight(i0 + k) * rstd;
        amax = fmaxf(amax, fabsf(y[k]));
      }
      amax = fmaxf(group_max<32>(amax), 1e-10f);
      const float s = __fdiv_rn(amax, 448.f);
      const Ue8m0 e = ue8m0_of(amax);
      const float inv = KIND == B200_ROW_FP8 ? __frcp_rn(s) : e.inv;
      const uint32_t out = pack4_e4m3(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
      *reinterpret_cast<uint32_t*>(p.q + row * H + i0) = out;
      if ((threadIdx.x & 31) == 0) put_group_scale<KIND>(p, row, g, s, e.byte);
    }
  }
}

template <typename T, int SRC, int KIND>
static int launch_rows(const RowParams& p, cudaStream_t st, const char* what) {
  return launch_dependent(row_quant_any_kernel<T, SRC, KIND>, dim3((unsigned)p.rows), 256, 0, st, 1, what, p);
}

template <int SRC, int KIND>
static int launch_rows(int dtype, const RowParams& p, cudaStream_t st, const char* what) {
  B200_UNSUPPORTED(p.rows > 0x7fffffffLL, "%s: more than 2^31 - 1 rows", what);
  switch (dtype) {
    case B200_BF16: return launch_rows<__nv_bfloat16, SRC, KIND>(p, st, what);
    case B200_F16: return launch_rows<__half, SRC, KIND>(p, st, what);
    default: return launch_rows<float, SRC, KIND>(p, st, what);
  }
}

}  // namespace b200

extern "C" int b200_rmsnorm_quant(const void* x, int64_t x_ld, const void* residual, int64_t residual_ld, const void* weight,
                                  int dtype, int kind, void* q, void* s, int64_t s_stride_m, int64_t s_stride_g,
                                  void* residual_out, int64_t M, int64_t H, float eps, void* stream) {
  using namespace b200;
  B200_CHECK_ARG(M >= 0 && H >= 0, "rmsnorm_quant: negative shape");
  B200_CHECK_ARG(dtype == B200_BF16 || dtype == B200_F16 || dtype == B200_F32, "rmsnorm_quant: unknown dtype code %d", dtype);
  B200_CHECK_ARG(kind == B200_ROW_INT8 || kind == B200_ROW_FP8 || kind == B200_ROW_FP8_UE8M0, "rmsnorm_quant: unknown kind %d", kind);
  if (M == 0 || H == 0) return B200_OK;
  B200_CHECK_ARG(x && weight && q && s, "rmsnorm_quant: null pointer");
  B200_CHECK_ARG((residual == nullptr) == (residual_out == nullptr), "rmsnorm_quant: the residual and its output go together");
  B200_CHECK_ARG(kind == B200_ROW_INT8 || H % 128 == 0, "rmsnorm_quant: H=%lld is not a multiple of the group of 128", (long long)H);
  B200_UNSUPPORTED(H > (1 << 24), "rmsnorm_quant: H=%lld", (long long)H);
  const size_t es = dtype == B200_F32 ? 4 : 2;
  B200_CHECK_ARG(((uintptr_t)x % es | (uintptr_t)residual % es | (uintptr_t)weight % es | (uintptr_t)residual_out % es) == 0 &&
                     (uintptr_t)q % (kind == B200_ROW_INT8 ? 1 : 16) == 0 && (uintptr_t)s % 4 == 0,
                 "rmsnorm_quant: misaligned pointer");
  RowParams p = {x, x_ld, residual, residual_ld, weight, residual_out, static_cast<uint8_t*>(q), s, s_stride_m, s_stride_g, M, (int)H, eps};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define B200_ROWS(SRC)                                                                                       \
  return kind == B200_ROW_INT8  ? launch_rows<SRC, B200_ROW_INT8>(dtype, p, st, "rmsnorm_quant")             \
         : kind == B200_ROW_FP8 ? launch_rows<SRC, B200_ROW_FP8>(dtype, p, st, "rmsnorm_quant")              \
                                : launch_rows<SRC, B200_ROW_FP8_UE8M0>(dtype, p, st, "rmsnorm_quant")
  if (residual) B200_ROWS(ROW_ADD_NORM);
  B200_ROWS(ROW_NORM);
#undef B200_ROWS
}

extern "C" int b200_per_token_quant_int8(const void* x, int64_t x_ld, int dtype, void* q, float* s, int64_t M, int64_t K,
                                         int fuse_silu_and_mul, void* stream) {
  using namespace b200;
  B200_CHECK_ARG(M >= 0 && K >= 0, "per_token_quant_int8: negative shape");
  B200_CHECK_ARG(dtype == B200_BF16 || dtype == B200_F16 || dtype == B200_F32, "per_token_quant_int8: unknown dtype code %d", dtype);
  if (M == 0 || K == 0) return B200_OK;
  B200_CHECK_ARG(x && q && s, "per_token_quant_int8: null pointer");
  B200_UNSUPPORTED(K > (1 << 24), "per_token_quant_int8: K=%lld", (long long)K);
  B200_CHECK_ARG((uintptr_t)x % (dtype == B200_F32 ? 4 : 2) == 0 && (uintptr_t)s % 4 == 0, "per_token_quant_int8: misaligned pointer");
  RowParams p = {x, x_ld, nullptr, 0, nullptr, nullptr, static_cast<uint8_t*>(q), s, 1, 0, M, (int)K, 0.f};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return fuse_silu_and_mul ? launch_rows<ROW_SILU, B200_ROW_INT8>(dtype, p, st, "per_token_quant_int8")
                           : launch_rows<ROW_PLAIN, B200_ROW_INT8>(dtype, p, st, "per_token_quant_int8");
}
