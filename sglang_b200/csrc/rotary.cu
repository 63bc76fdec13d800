// Heads of q, k and v between the qkv linear and attention, in one pass: RMSNorm of every head of q and k, rotation by position, q (and k) as
// new rows, or k and v into the pages of a cache, in 16 bits or in E4M3.
//   norm    y = x * w * rsqrt(mean(x^2) + eps) over a head's D elements
//   rotate  pair j of R / 2: (a, b) -> (a c - b s, b c + a s), c | s = row `position` of a table [positions, R]; a, b are elements j and j + R / 2,
//           or 2j and 2j + 1; elements from R on pass. With several axes every pair takes the row of its own axis' position.
//   hold    the cache's type, or e4m3(y / scale) by the IEEE quotient
// All in fp32 from the 16-bit input to the one rounding of the result: a 16-bit value between norm and rotation would add its half step.
#include <type_traits>

#include "int8_round.cuh"

namespace b200 {

struct RopeParams {
  b200_rope_args a;
  uint32_t axis_of[16];  // 2 bits per pair, 16 pairs a word
  int split;             // warps per token
  FastDiv split_div;
  int per_warp;          // heads of one of them
  int page_shift;        // log2 of the page size, -1: not a power of two
};

constexpr int kRopePairs = 256;  // 512 rotated elements at most, by the bits of axis_of

__device__ __forceinline__ int64_t load_index(const void* p, int dtype, int64_t i) {
  return dtype == B200_I64 ? static_cast<const volatile int64_t*>(p)[i] : (int64_t)static_cast<const volatile int32_t*>(p)[i];
}

// The table's row of an axis, null where the position is outside the table: such tokens become NaN instead of reading elsewhere.
__device__ __forceinline__ const float* table_row(const b200_rope_args& a, int axis, int64_t row) {
  const int64_t at = load_index(a.positions, a.positions_dtype, axis * a.positions_ld + row);
  return at >= 0 && at < a.table_rows ? a.cos_sin + at * a.cos_sin_ld : nullptr;
}
__device__ __forceinline__ int axis_of_pair(const RopeParams& p, int j) { return (p.axis_of[j >> 4] >> (2 * (j & 15))) & 3; }

// Where a token's keys and values go: element offsets of its row in the two caches; false where the slot is none of the cache's.
struct SlotAt {
  int64_t k, v;
};
__device__ __forceinline__ bool slot_at(const RopeParams& p, int64_t row, SlotAt& at) {
  const b200_rope_args& a = p.a;
  const int64_t slot = load_index(a.slots, a.slots_dtype, row);
  if (slot < 0 || slot >= a.pages * a.page_size) return false;
  const int64_t page = p.page_shift >= 0 ? slot >> p.page_shift : slot / a.page_size;
  const int64_t in_page = slot - page * a.page_size;
  at.k = page * a.k_cache_page + in_page * a.k_cache_token;
  at.v = page * a.v_cache_page + in_page * a.v_cache_token;
  return true;
}

// x / s as IEEE rounds it, r = 1 / s. Where the residual step has infinities in it, or has lost the sign of a zero, the product says it all.
__device__ __forceinline__ float scaled(float x, float s, float r) {
  const float q = div_by(x, s, r);
  return fabsf(q) > 0.f ? q : x * r;
}

// The reciprocal of a scale this small may be infinite: divisor and dividend go up by kLift, exactly, or to an infinity that saturates like the quotient.
constexpr float kSmallScale = 0x1p-60f, kLift = 0x1p64f;

enum HeadKind { HEAD_Q = 0, HEAD_K = 1, HEAD_V = 2 };

// Two fp32 values in one register pair, and the operations that take both at once: half the instructions of the norm and the rotation.
struct Two {
  uint64_t v;
  __device__ __forceinline__ Two() = default;
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ float2 get() const {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
  }
};
__device__ __forceinline__ Two mul(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// Two 16-bit values of a word, lowest first, and back
template <typename T>
__device__ __forceinline__ Two widen(uint32_t w) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) return Two(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return Two(f.x, f.y);
}
template <typename T>
__device__ __forceinline__ uint32_t narrow(Two t) {
  const float2 f = t.get();
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 r = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

// LANES lanes of a warp per head, two vectors of eight elements per lane. Elements j and j + R / 2 of a pair lie in the lane's two vectors
// (NEOX), or pairs lie within a vector. A warp takes 32 / LANES heads of one token at a time, UNROLL times that are under way together, first those of q, then
// of k, then of v; the angles stay in its registers for all of them.
// Bound by the latency between a token's position, its angles and its heads, so what counts are heads under way: 80 registers and two steps a warp hide more than
// 124 and four (16384 x 72 heads of 128, three axes: 129 us, 4.75 TB/s, against 133; into an FP8 cache, 8192 x 48: 57 against 63), 64 registers or asking
// for all steps of a batch after the last of the one before less (156, 150): in a graph, caches cold. Calls one after another take 133 and 53.
template <typename T, int LANES, bool NEOX, int UNROLL>
__global__ void __launch_bounds__(256, 3) rope_heads_kernel(const __grid_constant__ RopeParams p) {
  const b200_rope_args& a = p.a;
  grid_launch_dependents();
  const int64_t zero = grid_dependency_zero();
  const int warp = (int)(blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5));
  const int64_t row = fast_div(warp, p.split_div) + zero;
  if (row >= a.rows) return;
  constexpr int kTeams = 32 / LANES;
  const int lane = threadIdx.x % LANES, team = (threadIdx.x & 31) / LANES;
  const int nvec = a.dim >> 3, P = NEOX ? a.rotated >> 4 : 0, rest = (nvec - 2 * P + 1) >> 1;
  const bool turned = lane < P;  // (NEOX)
  const int va = turned ? lane : lane + P, vb = turned ? lane + P : va + rest;
  const bool has_a = lane < P + rest, has_b = has_a && vb < nvec;
  const int nq = a.q ? a.q_heads : 0, nk = a.k ? a.kv_heads : 0, total = nq + nk + (a.v ? a.kv_heads : 0);
  const int first = (warp - (int)row * p.split) * p.per_warp, last = min(first + p.per_warp, total);

  auto load = [&](const T* src, int h, int end, uint4 (&x)[2]) {
    x[0] = x[1] = make_uint4(0, 0, 0, 0);
    if (h < end && has_a) x[0] = ld_stream_16(src + va * 8);
    if (h < end && has_b) x[1] = ld_stream_16(src + vb * 8);
  };
  // NEOX: c, s of pairs 8 lane .. 8 lane + 7; else of pairs 4 va .. and 4 vb ..
  float c[8], s[8];
  auto load_angles = [&] {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
    if (a.rotated == 0) return;
    const int pairs = a.rotated >> 1;
    const float* rows[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) rows[k] = k < a.axes ? table_row(a, k, row) : nullptr;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int j0 = NEOX ? lane * 8 + half * 4 : (half ? vb : va) * 4;
      if (NEOX ? turned : j0 < pairs) {
        if (a.axes == 1) {
          if (rows[0]) {
            const float4 cc = ld_operand(reinterpret_cast<const float4*>(rows[0] + j0));
            const float4 ss = ld_operand(reinterpret_cast<const float4*>(rows[0] + pairs + j0));
            c[half * 4] = cc.x, c[half * 4 + 1] = cc.y, c[half * 4 + 2] = cc.z, c[half * 4 + 3] = cc.w;
            s[half * 4] = ss.x, s[half * 4 + 1] = ss.y, s[half * 4 + 2] = ss.z, s[half * 4 + 3] = ss.w;
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) c[half * 4 + i] = s[half * 4 + i] = NAN;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int axis = axis_of_pair(p, j0 + i);
            const float* r = axis == 0 ? rows[0] : axis == 1 ? rows[1] : axis == 2 ? rows[2] : rows[3];
            c[half * 4 + i] = r ? ld_operand(r + j0 + i) : NAN;
            s[half * 4 + i] = r ? ld_operand(r + pairs + j0 + i) : NAN;
          }
        }
      }
    }
  };
  SlotAt at = {0, 0};
  const bool cached = a.k_cache != nullptr;
  bool keep = false, placed = false, angled = false;

  // The heads [lo, hi) of one kind that are this warp's
  auto heads = [&](auto kind_of, const void* from, int64_t token, int64_t head, const void* norm, int lo, int hi) {
    constexpr int kind = decltype(kind_of)::value;
    if (lo >= hi) return;
    const T* const src = static_cast<const T*>(from) + row * token + zero;
    const bool normed = kind != HEAD_V && norm != nullptr;
    uint4 x[UNROLL][2];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) load(src + (lo + u * kTeams + team) * head, lo + u * kTeams + team, hi, x[u]);
    Two w[8];
    if (normed) {
      uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
      const T* const weights = static_cast<const T*>(norm) + zero;
      if (has_a) raw[0] = ld_again_16(weights + va * 8);
      if (has_b) raw[1] = ld_again_16(weights + vb * 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = widen<T>(reinterpret_cast<const uint32_t*>(raw)[i]);
    }
    if (kind != HEAD_V && !angled) {
      load_angles();
      angled = true;
    }
    if (kind != HEAD_Q && cached && !placed) {
      keep = slot_at(p, row, at);
      placed = true;
    }
    const bool to_cache = kind != HEAD_Q && cached;
    const float* const scales = to_cache && a.cache_dtype == B200_E4M3 ? (kind == HEAD_K ? a.k_scale : a.v_scale) : nullptr;
    const bool one_scale = (kind == HEAD_K ? a.k_scales : a.v_scales) <= 1;

    auto finish = [&](int h, const uint4 (&v)[2]) {
      const uint32_t* words = reinterpret_cast<const uint32_t*>(v);
      if (kind == HEAD_V && !(to_cache && a.cache_dtype == B200_E4M3)) {  // copied
        if (h >= hi || !has_a || !keep) return;
        T* dst = static_cast<T*>(a.v_cache) + at.v + h * a.v_cache_head;
        *reinterpret_cast<uint4*>(dst + va * 8) = v[0];
        if (has_b) *reinterpret_cast<uint4*>(dst + vb * 8) = v[1];
        return;
      }
      Two f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = widen<T>(words[i]);
      if (normed) {  // every lane of the warp takes part in the sums
        Two sq = mul(f[0], f[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) sq = fma(f[i], f[i], sq);
        const float2 both = sq.get();
        float sum = both.x + both.y;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float r = __frsqrt_rn(sum / (float)a.dim + a.eps);
        const Two rr(r, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = mul(mul(f[i], rr), w[i]);
      }
      if (h >= hi || !has_a) return;
      if (kind != HEAD_V) {
        if constexpr (NEOX) {
          if (turned) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const Two e = f[i], o = f[i + 4], cc(c[2 * i], c[2 * i + 1]), ss(s[2 * i], s[2 * i + 1]), minus(-s[2 * i], -s[2 * i + 1]);
              f[i] = fma(o, minus, mul(e, cc));
              f[i + 4] = fma(e, ss, mul(o, cc));
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if ((i < 4 ? va : vb) * 8 >= a.rotated) continue;  // elements that pass keep their bits beside an infinity
            const float2 e = f[i].get();
            f[i] = Two(e.x * c[i] - e.y * s[i], e.y * c[i] + e.x * s[i]);
          }
        }
      }
      if (to_cache && a.cache_dtype == B200_E4M3) {
        if (!keep) return;
        float y[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 e = f[i].get();
          y[2 * i] = e.x, y[2 * i + 1] = e.y;
        }
        if (scales) {
          float d = ld_operand(scales + (one_scale ? 0 : h));
          if (fabsf(d) < kSmallScale) {
            d *= kLift;
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] *= kLift;
          }
          const float r = __frcp_rn(d);
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = scaled(y[i], d, r);
        }
        uint8_t* dst = kind == HEAD_K ? static_cast<uint8_t*>(a.k_cache) + at.k + h * a.k_cache_head : static_cast<uint8_t*>(a.v_cache) + at.v + h * a.v_cache_head;
        *reinterpret_cast<uint2*>(dst + va * 8) = make_uint2(pack4_e4m3(y[0], y[1], y[2], y[3]), pack4_e4m3(y[4], y[5], y[6], y[7]));
        if (has_b)
          *reinterpret_cast<uint2*>(dst + vb * 8) = make_uint2(pack4_e4m3(y[8], y[9], y[10], y[11]), pack4_e4m3(y[12], y[13], y[14], y[15]));
        return;
      }
      if (to_cache && !keep) return;
      T* dst = kind == HEAD_Q ? static_cast<T*>(a.q_out) + (row * a.q_heads + h) * a.dim
               : to_cache     ? static_cast<T*>(a.k_cache) + at.k + h * a.k_cache_head
                              : static_cast<T*>(a.k_out) + (row * a.kv_heads + h) * a.dim;
      *reinterpret_cast<uint4*>(dst + va * 8) = make_uint4(narrow<T>(f[0]), narrow<T>(f[1]), narrow<T>(f[2]), narrow<T>(f[3]));
      if (has_b) *reinterpret_cast<uint4*>(dst + vb * 8) = make_uint4(narrow<T>(f[4]), narrow<T>(f[5]), narrow<T>(f[6]), narrow<T>(f[7]));
    };
    // A head's place is asked for anew as soon as the one before it is done, so that UNROLL steps are always under way
    for (int h0 = lo; h0 < hi; h0 += UNROLL * kTeams) {
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int h = h0 + u * kTeams + team, next = h + UNROLL * kTeams;
        finish(h, x[u]);
        load(src + next * head, next, hi, x[u]);
      }
    }
  };
  heads(std::integral_constant<int, HEAD_Q>(), a.q, a.q_token, a.q_head, a.q_weight, min(first, nq), min(last, nq));
  heads(std::integral_constant<int, HEAD_K>(), a.k, a.k_token, a.k_head, a.k_weight, max(first - nq, 0), min(last - nq, nk));
  heads(std::integral_constant<int, HEAD_V>(), a.v, a.v_token, a.v_head, nullptr, max(first - nq - nk, 0), last - nq - nk);
}

// Any width, alignment and type: a warp per head, an element per lane at a time, read twice (once for the norm).
template <typename T>
__global__ void __launch_bounds__(256) rope_any_kernel(const __grid_constant__ RopeParams p) {
  const b200_rope_args& a = p.a;
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int nq = a.q ? a.q_heads : 0, nk = a.k ? a.kv_heads : 0, total = nq + nk + (a.v ? a.kv_heads : 0);
  const int64_t warp = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t row = warp / total;
  if (row >= a.rows) return;
  const int h = (int)(warp % total), kind = h < nq ? HEAD_Q : h < nq + nk ? HEAD_K : HEAD_V;
  const int g = kind == HEAD_Q ? h : kind == HEAD_K ? h - nq : h - nq - nk;
  const volatile T* x = static_cast<const T*>(kind == HEAD_Q ? a.q : kind == HEAD_K ? a.k : a.v) +
                        (kind == HEAD_Q ? row * a.q_token + g * a.q_head : kind == HEAD_K ? row * a.k_token + g * a.k_head
                                                                                          : row * a.v_token + g * a.v_head);
  const volatile T* w = static_cast<const T*>(kind == HEAD_Q ? a.q_weight : kind == HEAD_K ? a.k_weight : nullptr);
  auto element = [](const volatile T* q, int i) {
    if constexpr (sizeof(T) == 4) {
      return (float)q[i];
    } else {
      const uint16_t bits = reinterpret_cast<const volatile uint16_t*>(q)[i];
      return to_f32<T>(*reinterpret_cast<const T*>(&bits));
    }
  };
  float r = 1.f;
  if (w) {
    float sum = 0.f;
    for (int i = lane; i < a.dim; i += 32) {
      const float f = element(x, i);
      sum = fmaf(f, f, sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    r = __frsqrt_rn(sum / (float)a.dim + a.eps);
  }
  SlotAt at = {0, 0};
  const bool cached = a.k_cache != nullptr && kind != HEAD_Q;
  if (cached && !slot_at(p, row, at)) return;
  const int64_t to = kind == HEAD_K ? at.k + g * a.k_cache_head : at.v + g * a.v_cache_head;
  float d = 1.f, rd = 1.f, lift = 1.f;
  const float* scales = !cached ? nullptr : kind == HEAD_K ? a.k_scale : a.v_scale;
  if (scales) {
    d = ld_operand(scales + ((kind == HEAD_K ? a.k_scales : a.v_scales) > 1 ? g : 0));
    if (fabsf(d) < kSmallScale) lift = kLift;
    d *= lift;
    rd = __frcp_rn(d);
  }
  auto normed = [&](int i) {
    const float f = element(x, i);
    return w ? f * r * element(w, i) : f;
  };
  const int pairs = a.rotated >> 1;
  for (int i = lane; i < a.dim; i += 32) {
    float f = normed(i);
    if (kind != HEAD_V && i < a.rotated) {
      const int j = a.neox ? i % pairs : i >> 1;
      const bool second = a.neox ? i >= pairs : i & 1;
      const float other = normed(a.neox ? (second ? i - pairs : i + pairs) : i ^ 1);
      const float* line = table_row(a, a.axes == 1 ? 0 : axis_of_pair(p, j), row);
      const float c = line ? ld_operand(line + j) : NAN, s = line ? ld_operand(line + pairs + j) : NAN;
      f = second ? f * c + other * s : f * c - other * s;
    }
    if (!cached) {
      T* dst = kind == HEAD_Q ? static_cast<T*>(a.q_out) + (row * a.q_heads + g) * a.dim : static_cast<T*>(a.k_out) + (row * a.kv_heads + g) * a.dim;
      dst[i] = from_f32<T>(f);
    } else if (a.cache_dtype != B200_E4M3) {
      (static_cast<T*>(kind == HEAD_K ? a.k_cache : a.v_cache) + to)[i] = from_f32<T>(f);
    } else {
      (static_cast<uint8_t*>(kind == HEAD_K ? a.k_cache : a.v_cache) + to)[i] =
          (uint8_t)__nv_cvt_float_to_fp8(scales ? scaled(f * lift, d, rd) : f, __NV_SATFINITE, __NV_E4M3);
    }
  }
}

template <typename T, int LANES>
static int launch_heads(RopeParams& p, int total, cudaStream_t st) {
  constexpr int kTeams = 32 / LANES, kUnroll = 2;
  // Few tokens: a warp for every step of heads, so that all loads leave at once; many: a warp keeps a token's angles for all of its heads
  const int64_t steps = cdiv(total, kTeams);
  int64_t split = cdiv(148 * 32, p.a.rows);
  split = split > steps ? steps : split;
  p.per_warp = (int)cdiv(steps, split) * kTeams;
  p.split = (int)cdiv(total, p.per_warp);
  const unsigned threads = p.a.rows * p.split >= 148 * 8 ? 256 : 128;
  const int64_t blocks = cdiv(p.a.rows * p.split, threads / 32);
  B200_UNSUPPORTED(p.a.rows * p.split > 0x7ffffff0LL, "qk_norm_rope: too many rows");
  p.split_div = make_fastdiv(p.split);
  const dim3 grid((unsigned)blocks);
  return p.a.neox ? launch_dependent(rope_heads_kernel<T, LANES, true, kUnroll>, grid, threads, 0, st, 1, "qk_norm_rope", p)
                  : launch_dependent(rope_heads_kernel<T, LANES, false, kUnroll>, grid, threads, 0, st, 1, "qk_norm_rope", p);
}

template <typename T>
static int launch_rope(RopeParams& p, cudaStream_t st) {
  const b200_rope_args& a = p.a;
  const int total = (a.q ? a.q_heads : 0) + (a.k ? a.kv_heads : 0) + (a.v ? a.kv_heads : 0);
  if (total == 0) return B200_OK;
  // 16-byte vectors of elements and angles; pairs whose halves lie whole vectors apart
  auto rows16 = [](const void* q, int64_t token, int64_t head) { return !q || ((uintptr_t)q % 16 == 0 && token % 8 == 0 && head % 8 == 0); };
  const uintptr_t held = a.cache_dtype == B200_E4M3 ? 8 : 16;
  bool vectors = sizeof(T) == 2 && a.dim % 8 == 0 && a.dim <= 512 && a.rotated % (a.neox ? 16 : 8) == 0 && rows16(a.q, a.q_token, a.q_head) &&
                 rows16(a.k, a.k_token, a.k_head) && rows16(a.v, a.v_token, a.v_head) && rows16(a.q_weight, 0, 0) && rows16(a.k_weight, 0, 0) &&
                 rows16(a.q_out, 0, 0) && rows16(a.k_out, 0, 0) && (uintptr_t)a.cos_sin % 16 == 0 && a.cos_sin_ld % 4 == 0;
  if (a.k_cache)
    vectors = vectors && (uintptr_t)a.k_cache % held == 0 && (uintptr_t)a.v_cache % held == 0 &&
              (a.k_cache_page | a.k_cache_token | a.k_cache_head | a.v_cache_page | a.v_cache_token | a.v_cache_head) % 8 == 0;
  if constexpr (sizeof(T) == 2) {
    if (vectors) {
      const int lanes = (a.dim / 8 + 1) / 2;
      return lanes <= 4    ? launch_heads<T, 4>(p, total, st)
             : lanes <= 8  ? launch_heads<T, 8>(p, total, st)
             : lanes <= 16 ? launch_heads<T, 16>(p, total, st)
                           : launch_heads<T, 32>(p, total, st);
    }
  }
  const int64_t blocks = cdiv(a.rows * total, 8);
  B200_UNSUPPORTED(blocks > 0x7fffffffLL, "qk_norm_rope: too many rows");
  return launch_dependent(rope_any_kernel<T>, dim3((unsigned)blocks), 256, 0, st, 1, "qk_norm_rope", p);
}

}  // namespace b200

extern "C" int b200_qk_norm_rope(const b200_rope_args* args, void* stream) {
  using namespace b200;
  B200_CHECK_ARG(args != nullptr, "qk_norm_rope: null pointer");
  RopeParams p = {};
  p.a = *args;
  const b200_rope_args& a = p.a;
  B200_CHECK_ARG(a.rows >= 0 && a.q_heads >= 0 && a.kv_heads >= 0 && a.dim >= 0, "qk_norm_rope: negative shape");
  B200_CHECK_ARG(a.dtype == B200_BF16 || a.dtype == B200_F16 || a.dtype == B200_F32, "qk_norm_rope: unknown dtype code %d", a.dtype);
  B200_CHECK_ARG(a.rotated >= 0 && a.rotated % 2 == 0 && a.rotated <= a.dim, "qk_norm_rope: %d of %d elements cannot rotate", a.rotated, a.dim);
  B200_UNSUPPORTED(a.rotated > 2 * kRopePairs, "qk_norm_rope: more than %d rotated elements", 2 * kRopePairs);
  B200_UNSUPPORTED(a.dim > (1 << 20) || a.q_heads > (1 << 20) || a.kv_heads > (1 << 20), "qk_norm_rope: heads of this size");
  if (a.rows == 0 || a.dim == 0) return B200_OK;
  const bool cached = a.k_cache != nullptr;
  B200_CHECK_ARG((a.q == nullptr) == (a.q_out == nullptr) && (a.q || a.k) && (a.k == nullptr || cached || a.k_out),
                 "qk_norm_rope: null pointer");
  B200_CHECK_ARG(cached == (a.v_cache != nullptr) && cached == (a.slots != nullptr) && cached == (a.v != nullptr) && (!cached || a.k),
                 "qk_norm_rope: k, v, both caches and the slots go together");
  const int es = a.dtype == B200_F32 ? 4 : 2;
  B200_CHECK_ARG(((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.k_out | (uintptr_t)a.q_weight |
                  (uintptr_t)a.k_weight) % es == 0, "qk_norm_rope: misaligned pointer");
  if (cached) {
    B200_CHECK_ARG(a.cache_dtype == a.dtype || a.cache_dtype == B200_E4M3, "qk_norm_rope: the cache has the input's type or E4M3");
    B200_CHECK_ARG(a.cache_dtype == B200_E4M3 || ((uintptr_t)a.k_cache | (uintptr_t)a.v_cache) % es == 0, "qk_norm_rope: misaligned pointer");
    B200_CHECK_ARG(a.cache_dtype == B200_E4M3 || (!a.k_scale && !a.v_scale), "qk_norm_rope: scales belong to an E4M3 cache");
    B200_CHECK_ARG((!a.k_scale || a.k_scales == 1 || a.k_scales == a.kv_heads) && (!a.v_scale || a.v_scales == 1 || a.v_scales == a.kv_heads),
                   "qk_norm_rope: one scale, or one per head");
    B200_CHECK_ARG(a.page_size > 0 && a.pages >= 0 && (a.slots_dtype == B200_I32 || a.slots_dtype == B200_I64), "qk_norm_rope: pages or slots");
    p.page_shift = -1;
    for (int i = 0; i < 31; ++i)
      if (a.page_size == 1 << i) p.page_shift = i;
  }
  if (a.rotated > 0) {
    const int pairs = a.rotated / 2;
    B200_CHECK_ARG(a.positions && a.cos_sin && (uintptr_t)a.cos_sin % 4 == 0 && a.table_rows >= 0, "qk_norm_rope: positions and their table");
    B200_CHECK_ARG(a.positions_dtype == B200_I32 || a.positions_dtype == B200_I64, "qk_norm_rope: positions are int32 or int64");
    B200_CHECK_ARG(a.axes >= 1, "qk_norm_rope: %d axes", a.axes);
    B200_UNSUPPORTED(a.axes > 4, "qk_norm_rope: more than four axes");
    if (a.axes > 1) {
      int sum = 0;
      for (int k = 0; k < a.axes; ++k) {
        B200_CHECK_ARG(a.sections[k] >= 0, "qk_norm_rope: a negative section");
        sum += a.sections[k];
      }
      B200_CHECK_ARG(sum == pairs, "qk_norm_rope: the sections have %d pairs, the table %d", sum, pairs);
      int end = a.sections[0], run = 0;
      for (int j = 0; j < pairs; ++j) {
        int axis;
        if (a.sections_interleaved) {
          axis = j % a.axes;
          if (j >= a.axes * a.sections[axis]) axis = 0;
        } else {
          while (j >= end) end += a.sections[++run];
          axis = run;
        }
        p.axis_of[j >> 4] |= (uint32_t)axis << (2 * (j & 15));
      }
    }
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a.dtype) {
    case B200_BF16: return launch_rope<__nv_bfloat16>(p, st);
    case B200_F16: return launch_rope<__half>(p, st);
    default: return launch_rope<float>(p, st);
  }
}
