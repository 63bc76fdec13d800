// Rows of 16-bit (or fp32) activations -> 8-bit rows with scales, with what precedes the quantiser in a decoder layer fused in:
//   rmsnorm_quant          h = x (+ r);  y = h * w * rsqrt(mean(h^2) + eps);  r_out = h rounded once
//   per_token_quant_int8   y = x, or silu(gate) * up of rows [gate | up]
// and three ways to hold y in 8 bits:
//   int8      s = max|y| / 127 per row,               q = rint(y / s)
//   fp8       s = max|y| / 448 per 128 columns,       q = e4m3(y / s), fp32 scales with any strides
//   fp8 ue8m0 s = 2^ceil(log2(max|y| / 448)) likewise, exponent bytes packed four groups per int32 word, rows contiguous
// Sums and maxima are fp32; the floor of a maximum is 1e-10 as in the group quantiser. A row or group with a NaN in it gets a NaN
// (int8: as its scale, there is no NaN code; fp8: as codes).
// 1/rms cancels in y / s: the codes of a norm come from v = h * w and max|v|, so neither the order of the sum of squares nor, with it, the
// alignment and the number of the rows move them; only the scales (and power-of-two scales' codes) hold 1/rms.
#include <type_traits>

#include "int8_round.cuh"

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

// Sum and maximum over a row's threads (of a warp, or of the whole block); every thread gets both. red: 64 floats of shared memory.
template <bool SUM, bool MAX>
__device__ __forceinline__ void row_sum_max(float& sum, float& top, int warps, float* red) {
  auto warp_reduce = [&] {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (SUM) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (MAX) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
  };
  warp_reduce();
  if (warps == 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) {
    if (SUM) red[warp] = sum;
    if (MAX) red[32 + warp] = top;
  }
  __syncthreads();
  if (SUM) sum = lane < warps ? red[lane] : 0.f;
  if (MAX) top = lane < warps ? red[32 + lane] : 0.f;
  warp_reduce();
}

__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

constexpr float kFloor = 1e-10f;

// Scale of a row of 8-bit integers, and how its values v = y / rstd become codes, the nearest whole numbers (top = max|v|):
//   plain, norms  of the quotient v / step: of 16-bit inputs it is often an exact tie, which a rounded factor sends either way (8.4 million normed values:
//                 0.4 codes off the exact ones, 7 with a factor, 3 in the plain form)
//                 (203 x 8192 3.07 us, with a factor 2.97)
//   gated         of the product v * inv, inv = 127 / top rounded once: silu leaves no ties, and quotients cost 6 % (8192 x 14336 101 -> 108 us)
struct RowScale {
  float s, step, inv;
};
template <int SRC>
__device__ __forceinline__ RowScale int8_row_scale(float top, float rstd) {
  RowScale c;
  c.s = int8_scale(top * rstd);
  if constexpr (SRC == ROW_SILU) {
    c.step = 0.f;
    c.inv = __fdiv_rn(127.f, fmaxf(top, kFloor));
  } else {
    c.step = SRC == ROW_PLAIN ? c.s : top * rstd > kFloor ? over_127(top) : __fdiv_rn(kFloor / 127.f, rstd);
    c.inv = __frcp_rn(c.step);
    if (SRC != ROW_PLAIN && !(c.step < INFINITY)) c.step = c.inv = 0.f;  // a sum of squares past the largest float leaves y = 0
  }
  return c;
}

// The IEEE quotient: one residual step rounds it right for every mantissa
__device__ __forceinline__ float over_448(float m) { return m < INFINITY ? div_by(m, 448.f, 1.f / 448.f) : m; }

// Likewise of a group of FP8 values, code e4m3(v * factor). A power of two does not hold the maximum, so there the factor holds rstd.
// quotient: 448 / amax, which need not wait for rstd. With approximate quotients 203 x 4096 takes 2.94 us instead of 3.03, and more codes
// lie on the other side of a tie than in the plain form.
struct GroupScale {
  float top;      // s = top / 448
  uint32_t byte;  // ue8m0, by the group quantiser's arithmetic
  float factor;
};
template <int KIND>
__device__ __forceinline__ float fp8_quotient(float amax) { return KIND == B200_ROW_FP8 ? __fdiv_rn(448.f, amax) : 0.f; }
template <int KIND>
__device__ __forceinline__ GroupScale fp8_group_scale(float amax, float quotient, float rstd) {
  const float t = amax * rstd, m = fmaxf(t, kFloor);
  if constexpr (KIND == B200_ROW_FP8) {
    return {m, 0u, t > kFloor ? quotient : rstd * (448.f / kFloor)};
  } else {
    const uint32_t bits = __float_as_uint(m * (1.0f / 448.0f));
    const uint32_t byte = ((bits >> 23) & 0xffu) + ((bits & 0x7fffffu) != 0 ? 1u : 0u);
    return {m, byte, rstd * __uint_as_float((254u - byte) << 23)};
  }
}

template <int KIND>
__device__ __forceinline__ void put_group_scale(const RowParams& p, int64_t row, int g, const GroupScale& c) {
  if constexpr (KIND == B200_ROW_FP8) {
    static_cast<float*>(p.s)[row * p.s_sm + g * p.s_sg] = over_448(c.top);
  } else {
    uint8_t* dst = static_cast<uint8_t*>(p.s) + ((int64_t)(g >> 2) * p.s_sg + row) * 4 + (g & 3);
    *dst = (uint8_t)c.byte;
    if ((g + 1) * 128 == p.H)  // bytes of the last word that belong to no group read as zero
      for (int k = (g & 3) + 1; k < 4; ++k) dst[k - (g & 3)] = 0;
  }
}

// A row per block, element by element, some of them under way at once: any width and alignment. KEEP: the values wait in shared memory, as
// fp32, for the row's scale (gated 8192 x 5001 65 us, computed twice 79 with one element at a time, 112 with four). A plain row is read again
// instead, 43 against 45. Bound by the instructions per element: 2.8 to 3 TB/s.
constexpr int kKeepWidth = 12000;  // beside the reductions' 256 bytes it stays below the 48 KB of any launch
template <typename T, int SRC, int KIND, int BLOCK, bool KEEP>
__global__ void __launch_bounds__(BLOCK) row_quant_any_kernel(const RowParams p) {
  __shared__ float red[64];
  extern __shared__ float kept[];
  grid_dependency_wait();
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  const T* r = static_cast<const T*>(p.r) + row * p.r_ld;
  const T* w = static_cast<const T*>(p.w);
  const int H = p.H;
  constexpr int kAtOnce = SRC == ROW_PLAIN || SRC == ROW_NORM ? 8 : 4;  // elements under way
  auto value = [&](int i) {
    const float v = to_f32<T>(x[i]);
    if constexpr (SRC == ROW_SILU) return silu_mul(v, to_f32<T>(x[H + i]));
    if constexpr (SRC == ROW_ADD_NORM) return v + to_f32<T>(r[i]);
    return v;
  };
  auto weight = [&](int i) { return SRC >= ROW_NORM ? to_f32<T>(w[i]) : 1.f; };
  float sum = 0.f, top = 0.f;
  for (int i0 = threadIdx.x; i0 < H; i0 += kAtOnce * BLOCK) {
    float h[kAtOnce], y[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int i = i0 + u * BLOCK;
      h[u] = i < H ? value(i) : 0.f;
      if (KEEP || KIND == B200_ROW_INT8) y[u] = i < H ? h[u] * weight(i) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int i = i0 + u * BLOCK;
      sum = fmaf(h[u], h[u], sum);
      if (KIND == B200_ROW_INT8) top = max_nan(top, fabsf(y[u]));
      if (KEEP && i < H) kept[i] = y[u];
      if (SRC == ROW_ADD_NORM && i < H) static_cast<T*>(p.r_out)[row * H + i] = from_f32<T>(h[u]);
    }
  }
  row_sum_max<true, true>(sum, top, BLOCK / 32, red);
  const float rstd = SRC >= ROW_NORM ? rsqrtf(sum / (float)H + p.eps) : 1.f;
  auto weighted = [&](int i) { return KEEP ? kept[i] : value(i) * weight(i); };
  if constexpr (KIND == B200_ROW_INT8) {
    const RowScale c = int8_row_scale<SRC>(top, rstd);
    if (threadIdx.x == 0) static_cast<float*>(p.s)[row] = c.s;
    for (int i0 = threadIdx.x; i0 < H; i0 += kAtOnce * BLOCK) {
      float y[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int i = i0 + u * BLOCK;
        y[u] = i < H ? weighted(i) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (i0 + u * BLOCK < H)
          p.q[row * H + i0 + u * BLOCK] = (uint8_t)(SRC == ROW_SILU ? rint_scaled(y[u], c.inv) : rint_bits(div_by(y[u], c.step, c.inv)));
    }
  } else {  // 128 columns: four per lane of a warp
    for (int g = threadIdx.x >> 5; g * 128 < H; g += BLOCK / 32) {
      const int i0 = g * 128 + (threadIdx.x & 31) * 4;
      float y[4], amax = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        y[k] = weighted(i0 + k);
        amax = fmaxf(amax, fabsf(y[k]));
      }
      amax = group_max<32>(amax);
      const GroupScale c = fp8_group_scale<KIND>(amax, fp8_quotient<KIND>(amax), rstd);
      const uint32_t out = pack4_e4m3(y[0] * c.factor, y[1] * c.factor, y[2] * c.factor, y[3] * c.factor);
      *reinterpret_cast<uint32_t*>(p.q + row * H + i0) = out;
      if ((threadIdx.x & 31) == 0) put_group_scale<KIND>(p, row, g, c);
    }
  }
}

// Eight elements: what a thread loads at once
template <typename T>
struct Raw8 {
  static constexpr int kLoads = sizeof(T) * 8 / 16;
  uint4 v[kLoads];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) v[i] = ld_stream_16(p + i * (16 / sizeof(T)));
  }
  __device__ __forceinline__ void cached(const T* p) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) v[i] = ld_again_16(p + i * (16 / sizeof(T)));
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) v[i] = make_uint4(0, 0, 0, 0);
  }
  // largest magnitude, a NaN if there is one
  __device__ __forceinline__ float amax() const {
    if constexpr (sizeof(T) == 2) {
      using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
      const T2* p = reinterpret_cast<const T2*>(v);
      const T2 m = __hmax2_nan(__hmax2_nan(__habs2(p[0]), __habs2(p[1])), __hmax2_nan(__habs2(p[2]), __habs2(p[3])));
      return max_nan(to_f32<T>(m.x), to_f32<T>(m.y));
    } else {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(get(i)));
      return m;
    }
  }
  __device__ __forceinline__ float get(int i) const { return to_f32<T>(reinterpret_cast<const T*>(v)[i]); }
  __device__ __forceinline__ void set(int i, float f) { reinterpret_cast<T*>(v)[i] = from_f32<T>(f); }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) reinterpret_cast<uint4*>(p)[i] = v[i];
  }
};

// What counts for many rows are the rows in flight, as a block loads, then reduces, and only other blocks' loads keep the memory busy
// meanwhile: registers are held down (0: as the compiler sees fit; plain 16384 x 1024 9.2 -> 8.4 us at three blocks). For few rows it is a
// block's own latency: `ahead`, the norm's weights are requested together with the row, whatever registers that takes.
constexpr int row_min_blocks(int src, int vpt, bool ahead) {
  return ahead || vpt > 4 ? 1 : src == ROW_SILU ? 2 : src == ROW_PLAIN && vpt == 4 ? 3 : 0;
}

// A row in the registers of a block, or of a warp (blockDim.y rows per block): one pass over memory. A thread has VPT vectors of eight
// elements, blockDim.x vectors apart, so loads are 16 bytes per lane without gaps, and all of them are under way before the
// first is used.
template <typename T, int SRC, int KIND, int VPT, bool AHEAD>
__global__ void __launch_bounds__(VPT <= 2 ? 1024 : 512, row_min_blocks(SRC, VPT, AHEAD)) row_quant_kernel(const RowParams p) {
  constexpr bool kNorm = SRC >= ROW_NORM, kTwo = SRC == ROW_SILU || SRC == ROW_ADD_NORM;
  __shared__ float red[64];
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= p.rows) return;  // a whole warp: several rows to a block only where each has one
  const int H = p.H, nvec = H >> 3;
  grid_launch_dependents();
  const int64_t zero = grid_dependency_zero();
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld + zero;
  const T* second = SRC == ROW_SILU ? x + H : static_cast<const T*>(p.r) + row * p.r_ld + zero;
  const T* weight = static_cast<const T*>(p.w) + zero;
  Raw8<T> a[VPT], b[kTwo ? VPT : 1];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int v = threadIdx.x + j * blockDim.x;
    if (v < nvec) {
      a[j].load(x + v * 8);
      if (kTwo) b[j].load(second + v * 8);
    } else {
      a[j].zero();
      if (kTwo) b[j].zero();
    }
  }
  Raw8<T> w[kNorm && AHEAD ? VPT : 1];
  auto load_weights = [&](int j, Raw8<T>& to) {
    const int v = threadIdx.x + j * blockDim.x;
    if (v < nvec) to.cached(weight + v * 8);
    else to.zero();
  };
  if constexpr (kNorm && AHEAD) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) load_weights(j, w[j]);
  }
  // y as it is quantised; a plain row stays in its own type and is converted twice instead, which leaves registers for more rows
  float y[SRC == ROW_PLAIN ? 1 : VPT][8], sum = 0.f, top = 0.f;
  float amax[KIND == B200_ROW_INT8 ? 1 : VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    if constexpr (SRC == ROW_PLAIN) {
      top = max_nan(top, a[j].amax());
      continue;
    }
    const int v = threadIdx.x + j * blockDim.x;
    if (kNorm && !AHEAD) load_weights(j, w[0]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float h = a[j].get(i);
      if (SRC == ROW_SILU) h = silu_mul(h, b[j].get(i));
      if (SRC == ROW_ADD_NORM) {
        h += b[j].get(i);
        a[j].set(i, h);
      }
      if (kNorm) {
        sum = fmaf(h, h, sum);
        h *= w[AHEAD ? j : 0].get(i);
      }
      y[j][i] = h;
      if constexpr (KIND == B200_ROW_INT8) top = max_nan(top, fabsf(h));
    }
    if (SRC == ROW_ADD_NORM && v < nvec) a[j].store(static_cast<T*>(p.r_out) + row * H + v * 8);
    if constexpr (KIND != B200_ROW_INT8) {
      amax[j] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) amax[j] = fmaxf(amax[j], fabsf(y[j][i]));
    }
  }
  // 16 lanes hold VPT groups of 128 columns, one per vector: each step halves the values a lane still has, so that lane l ends with the
  // maximum, and then the scale, of group l % VPT (16384 x 8192 144 us, with every group's maximum and scale in every lane 153)
  if constexpr (KIND != B200_ROW_INT8) {
    int n = VPT;
#pragma unroll
    for (int bit = 1; bit < 16; bit <<= 1) {
      const bool upper = (threadIdx.x & bit) != 0;
      if (n > 1) {
        n /= 2;
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const float other = __shfl_xor_sync(0xffffffffu, upper ? amax[2 * i] : amax[2 * i + 1], bit);
          amax[i] = fmaxf(upper ? amax[2 * i + 1] : amax[2 * i], other);
        }
      } else {
        amax[0] = fmaxf(amax[0], __shfl_xor_sync(0xffffffffu, amax[0], bit));
      }
    }
  }
  const float quotient = fp8_quotient<KIND>(amax[0]);  // (amax: one unused value where the codes are int8)
  row_sum_max<kNorm, KIND == B200_ROW_INT8>(sum, top, blockDim.x >> 5, red);
  const float rstd = kNorm ? rsqrtf(sum / (float)H + p.eps) : 1.f;
  if constexpr (KIND == B200_ROW_INT8) {
    const RowScale scale = int8_row_scale<SRC>(top, rstd);
    const DivTwo div(scale.step, scale.inv);
    if (threadIdx.x == 0) static_cast<float*>(p.s)[row] = scale.s;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int v = threadIdx.x + j * blockDim.x;
      uint32_t c[8];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        if constexpr (SRC == ROW_PLAIN) div.rint_bits(a[j].get(i), a[j].get(i + 1), c[i], c[i + 1]);
        if constexpr (SRC == ROW_SILU) rint_scaled_two(y[j][i], y[j][i + 1], twice(scale.inv), c[i], c[i + 1]);
        if constexpr (kNorm) div.rint_bits(y[j][i], y[j][i + 1], c[i], c[i + 1]);
      }
      if (v < nvec) *reinterpret_cast<uint2*>(p.q + row * H + v * 8) = pack8_s8(c);
    }
  } else {
    const GroupScale c = fp8_group_scale<KIND>(amax[0], quotient, rstd);
    const int own = threadIdx.x & 15, first = (threadIdx.x & ~15) + own * blockDim.x;
    if (own < VPT && first < nvec) put_group_scale<KIND>(p, row, first >> 4, c);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int v = threadIdx.x + j * blockDim.x;
      const float f = __shfl_sync(0xffffffffu, c.factor, j, 16);
      uint2 out;
      out.x = pack4_e4m3(y[j][0] * f, y[j][1] * f, y[j][2] * f, y[j][3] * f);
      out.y = pack4_e4m3(y[j][4] * f, y[j][5] * f, y[j][6] * f, y[j][7] * f);
      if (v < nvec) *reinterpret_cast<uint2*>(p.q + row * H + v * 8) = out;
    }
  }
}

template <typename T, int SRC, int KIND, int VPT, bool AHEAD = false>
static int launch_row_regs(const RowParams& p, unsigned threads, unsigned rows_per_block, cudaStream_t st, const char* what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cdiv(p.rows, rows_per_block));
  cfg.blockDim = dim3(threads, rows_per_block);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, row_quant_kernel<T, SRC, KIND, VPT, AHEAD>, p);
  if (e != cudaSuccess) {
    set_error_detail("%s: %s", what, cudaGetErrorString(e));
    return B200_E_LAUNCH;
  }
  return check_launch(what);
}

template <typename T, int SRC, int KIND>
static int launch_rows(const RowParams& p, cudaStream_t st, const char* what) {
  // 16-byte loads and 8-byte stores, all of a row in registers
  const int64_t nvec = p.H / 8;
  auto even = [](const void* q, int64_t ld) { return (uintptr_t)q % 16 == 0 && ld * (int64_t)sizeof(T) % 16 == 0; };
  const bool vectors = p.H % 8 == 0 && nvec <= 4096 && (p.rows == 1 || p.x_ld % (16 / (int)sizeof(T)) == 0) && (uintptr_t)p.x % 16 == 0 &&
                       (SRC != ROW_ADD_NORM || (even(p.r, p.rows == 1 ? 0 : p.r_ld) && (uintptr_t)p.r_out % 16 == 0)) &&
                       (uintptr_t)p.w % 16 == 0 && (uintptr_t)p.q % 8 == 0;
  if (!vectors) {
    const dim3 grid((unsigned)p.rows);
    const size_t keep = (size_t)p.H * 4;
    constexpr bool kKeep = SRC != ROW_PLAIN;
    if (p.H <= 1024)  // 16384 x 701: 18 us; with 256 threads, an element at a time, 39
      return launch_dependent(row_quant_any_kernel<T, SRC, KIND, 128, kKeep>, grid, 128, kKeep ? keep : 0, st, 1, what, p);
    if (kKeep && p.H <= kKeepWidth)
      return launch_dependent(row_quant_any_kernel<T, SRC, KIND, 256, kKeep>, grid, 256, keep, st, 1, what, p);
    return launch_dependent(row_quant_any_kernel<T, SRC, KIND, 256, false>, grid, 256, 0, st, 1, what, p);
  }
  // us in a graph for 1 / 2 / 4 / 8 vectors a thread, 203 and 16384 rows of 8192 bf16:
  //   plain  2.4 / 2.8 / 3.2 / 3.2, 125 / 77 / 62 / 61 (6.6 TB/s)           gated  3.0 / 4.5 / 4.4 / 5.0, 135 / 112 / 106 / 132 (6.3)
  // norms with a residual for 1 / 2 / 4, the first two with `ahead`:
  //   203 x 8192   FP8 3.6 / 3.0 / 4.7, int8 3.8 / 3.1 / 4.9         8192 x 8192  FP8 88 / 81 / 74 (6.4 TB/s), int8 92 / 83 / 72 (6.5)
  //   2048 x 4096  FP8 11.0 / 9.1 / 10.3, int8 11.6 / 9.4 / 10.4     8192 x 4096  FP8 42 / 37 / 39, int8 43 / 37 / 39
  // Blocks that go through many rows, with a ring of them in shared memory that bulk copies fill, were no faster (plain 69 to 73 us).
  const bool short_or_few = nvec <= 512 || (p.rows <= 512 && nvec <= 1024);
  int vpt = SRC == ROW_PLAIN ? 8 : SRC == ROW_SILU ? (p.rows < 1024 ? 1 : 4) : short_or_few ? 2 : 4;
  if (tuning().row_vectors > 0) vpt = tuning().row_vectors < 8 ? (int)tuning().row_vectors : 8;
  while (vpt > 1 && nvec < 32 * vpt) vpt /= 2;
  while (vpt < 8 && cdiv(nvec, vpt) > (vpt <= 2 ? 1024 : 512)) vpt *= 2;
  const unsigned threads = (unsigned)align_up(cdiv(nvec, vpt), 32), rpb = threads == 32 ? 4 : 1;
  constexpr bool kNorm = SRC >= ROW_NORM;
  switch (vpt) {
    case 1: return launch_row_regs<T, SRC, KIND, 1, kNorm>(p, threads, rpb, st, what);
    case 2: return launch_row_regs<T, SRC, KIND, 2, kNorm>(p, threads, rpb, st, what);
    case 4: return launch_row_regs<T, SRC, KIND, 4>(p, threads, rpb, st, what);
    default: return launch_row_regs<T, SRC, KIND, 8>(p, threads, rpb, st, what);
  }
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
