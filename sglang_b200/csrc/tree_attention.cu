// Attention of the newest tokens of every sequence (one, or a tree of drafted ones) over a paged cache:
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale * k_scale * log2(e),  m near the largest exponent so far
// Query row r of a kv head is (token r / G, head r % G of the G query heads that share it); 128 rows are a tile of the tensor core's lanes, so that a
// softmax row belongs to one thread and needs no exchange, and few rows cost no more than the lanes they leave idle: bound by the cache's
// bytes, a tile of keys has more time than its two products and its exponentials take.
//   S [128, keys] = Q K^T        Q and K in shared memory, S in TMEM, two buffers
//   O [128, D]   += P V          P in TMEM over its own S, in the input's 16-bit type, V in shared memory as it lies in the cache
// Keys come by their pages' addresses, any page size, in 16-byte pieces by asynchronous copies (an FP8 cache through registers, where codes become
// 16-bit values, exactly). All tiles of all (sequence, kv head, row tile) form one line that is cut into equal pieces, one per CTA, so that ragged
// lengths leave no SM idle; rows whose keys were cut leave partial sums in a workspace, which a second kernel joins in the line's order.
#include "gemm_host.cuh"
#include "int8_round.cuh"

namespace b200 {
namespace ptx {

// D (+)= A B with 16-bit operands, fp32 sums; A in shared memory, or in TMEM (two elements a column)
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}" ::"r"(d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}" ::"r"(d),
      "r"(a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor for kind::f16, fp32 sums: bits 4-5 D format (1 = f32), 7-9 / 10-12 A / B format (0 = f16, 1 = bf16), 16 B is MN-major,
// 17-22 N >> 3, 24-28 M >> 4
__host__ __device__ constexpr uint32_t idesc_f16_f32(bool bf16, bool b_mn_major, int M, int N) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}
// Operand whose rows are k and whose 128-byte rows are 64 elements of N, 128-byte swizzle: 8-row groups 1024 bytes apart, the next 64 elements of N
// `block` bytes further
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t addr, uint32_t block) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(block >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}
// 16 columns of this thread's lane
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
      "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 16 bytes, or zeros (bytes = 0: nothing is read)
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void st_shared_16(uint32_t dst, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
}  // namespace ptx

// Rows whose keys were cut between CTAs: from the CTA where they begin, to the last one with a piece of them. parts == 0: none begin here.
struct SplitRows {
  int token, qt, head, rows, parts;
};

struct AttnParams {
  b200_tree_attention_args a;
  FastDiv group_div, page_div;
  int group;
  int row_slots;       // rows of a partial's slot
  float scale_log2;
  int64_t capacity;    // tokens that a sequence's line of the page table can name
  float* part_o;       // [2 grid][row_slots][D]
  float2* part_ml;     // [2 grid][row_slots]: reference of the exponents, sum
  SplitRows* split;    // [grid]
  int* status;
};

template <int D, bool FP8>
struct AttnCfg {
  static constexpr int kKeys = D > 128 ? 64 : 128;      // of a tile
  static constexpr int kStage = kKeys * D * 2;          // bytes of a tile of keys or values
  static constexpr int kQBytes = 128 * D * 2;
  static constexpr int kStages = D == 64 ? 10 : D == 128 ? 6 : 5;
  static constexpr int kAhead = 3;                      // stages whose copies are under way when the one before them is handed over
  static constexpr int kSoftmaxWarps = 4, kMmaWarp = 4, kQWarp = 5, kProducerWarp = 6, kProducerWarps = 4;
  static constexpr int kThreads = (kProducerWarp + kProducerWarps) * 32;
  static constexpr int kTmemO = 256;                    // columns: S 0 .. 2 kKeys, O from here
  static constexpr size_t kSmemBytes = (size_t)kQBytes + (size_t)kStages * kStage + 1024 + 512;
};

// Sequence b as the kernel takes it: whatever the index tensors hold, tokens and keys stay inside q and the page table.
struct Seq {
  int start, n, len, row_tiles, key_tiles;
  __device__ __forceinline__ int64_t tiles(int heads) const { return n > 0 ? (int64_t)heads * row_tiles * key_tiles : 0; }
};
template <int KEYS>
__device__ __forceinline__ Seq seq_of(const AttnParams& p, int b) {
  const b200_tree_attention_args& a = p.a;
  Seq s;
  int end;
  if (a.q_starts) {
    s.start = min(max(ld_operand(a.q_starts + b), 0), (int)a.tokens);
    end = min(max(ld_operand(a.q_starts + b + 1), s.start), (int)a.tokens);
  } else {
    s.start = min(b, (int)a.tokens);
    end = min(b + 1, (int)a.tokens);
  }
  s.n = end - s.start;
  s.len = (int)min((int64_t)max(ld_operand(a.seq_lens + b), 0), p.capacity);
  s.row_tiles = (s.n * p.group + 127) >> 7;
  s.key_tiles = max(1, (s.len + KEYS - 1) / KEYS);
  return s;
}

// A CTA's piece of the line, one (sequence, head, row tile) at a time
template <int KEYS>
struct Walk {
  const AttnParams& p;
  int b, h, qt, t0, t1;
  int64_t left;
  Seq s;
  __device__ __forceinline__ Walk(const AttnParams& p_, int b0, int64_t offset, int64_t count) : p(p_), b(b0), left(count) {
    h = qt = t0 = t1 = 0;
    s = {};
    if (left <= 0) return;
    s = seq_of<KEYS>(p, b);
    const int64_t per_head = (int64_t)s.row_tiles * s.key_tiles;
    h = (int)(offset / per_head);
    const int rest = (int)(offset - h * per_head);
    qt = rest / s.key_tiles;
    t0 = rest - qt * s.key_tiles;
    t1 = (int)min((int64_t)s.key_tiles, t0 + left);
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ void next() {
    left -= t1 - t0;
    if (left <= 0) return;
    t0 = 0;
    if (++qt == s.row_tiles) {
      qt = 0;
      if (++h == p.a.kv_heads) {
        h = 0;
        do {
          s = seq_of<KEYS>(p, ++b);
        } while (s.n == 0 && b + 1 < p.a.sequences);
      }
    }
    t1 = (int)min((int64_t)s.key_tiles, left);
  }
};

// Two E4M3 codes as 16-bit values: exact, both types hold all of them
template <typename T>
__device__ __forceinline__ uint32_t widen2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
  if constexpr (std::is_same_v<T, __half>) {
    return (uint32_t)h.x | ((uint32_t)h.y << 16);
  } else {
    const float2 f = __half22float2(__half2(h));
    const __nv_bfloat162 r = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

// References of the exponents may lie this far (in powers of two) below the largest: the sums stay exact to fp32 and P far from the 16-bit types'
// limits, and O is rescaled a few times per row instead of once per tile.
constexpr float kSlack = 8.f;

template <typename T, int D, bool FP8>
__global__ void __launch_bounds__(AttnCfg<D, FP8>::kThreads, 1) tree_attention_kernel(const __grid_constant__ AttnParams p) {
  using Cfg = AttnCfg<D, FP8>;
  constexpr int S = Cfg::kStages, KEYS = Cfg::kKeys;
  const b200_tree_attention_args& a = p.a;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_al = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
  const uint32_t sQ = smem_base, sKV = smem_base + Cfg::kQBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_al + Cfg::kQBytes + S * Cfg::kStage);
  const uint32_t bar0 = ptx::smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (S + s); };
  const uint32_t q_full = bar0 + 8u * (2 * S), q_empty = q_full + 8u, o_done = q_full + 16u;
  auto s_full = [&](int i) { return q_full + 24u + 8u * i; };
  auto p_full = [&](int i) { return q_full + 40u + 8u * i; };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(bars + 2 * S + 7);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * S + 8);
  volatile int* begin_seq = abort_flag + 1;
  volatile int64_t* line = reinterpret_cast<volatile int64_t*>(bars + 2 * S + 9);  // offset within the first sequence, tiles of this CTA, of every CTA
  volatile int64_t* sums = line + 3;                                               // of each warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      ptx::mbar_init(full_bar(s), Cfg::kProducerWarps);
      ptx::mbar_init(empty_bar(s), 1);
    }
    ptx::mbar_init(q_full, 1);
    ptx::mbar_init(q_empty, 1);
    ptx::mbar_init(o_done, 1);
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(s_full(i), 1);
      ptx::mbar_init(p_full(i), Cfg::kSoftmaxWarps);
    }
    *abort_flag = 0;
    *begin_seq = 0;
    line[0] = line[1] = 0;
    line[2] = 1;
    ptx::fence_mbar_init();
  }
  if (warp == Cfg::kMmaWarp) {
    ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_dependency_wait();

  // Where this CTA's piece begins: every thread adds up some consecutive sequences, the one whose part holds the beginning finds it
  {
    const int per = (int)((a.sequences + Cfg::kThreads - 1) / Cfg::kThreads);
    const int b0 = min((int)threadIdx.x * per, (int)a.sequences), b1 = min(b0 + per, (int)a.sequences);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += seq_of<KEYS>(p, b).tiles(a.kv_heads);
    int64_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t other = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += other;
    }
    if (lane == 31) sums[warp] = before;
    before -= mine;
    __syncthreads();
    int64_t total = 0;
    for (int w = 0; w < Cfg::kThreads / 32; ++w) {
      const int64_t v = sums[w];
      before += w < warp ? v : 0;
      total += v;
    }
    const int64_t chunk = max((total + gridDim.x - 1) / gridDim.x, (int64_t)1), begin = blockIdx.x * chunk;
    if (begin >= before && begin < before + mine) {
      for (int b = b0; b < b1; ++b) {
        const int64_t n = seq_of<KEYS>(p, b).tiles(a.kv_heads);
        if (begin < before + n) {
          *begin_seq = b;
          line[0] = begin - before;
          line[1] = min(chunk, total - begin);
          line[2] = chunk;
          break;
        }
        before += n;
      }
    }
    __syncthreads();
  }
  Walk<KEYS> w(p, *begin_seq, line[0], line[1]);
  const uint32_t lane_base = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
  bool ok = true;

  if (warp >= Cfg::kProducerWarp) {
    // ------------------------------------------------------------------ keys and values into the ring: K, V, K, V, ..
    constexpr int kRows = KEYS / Cfg::kProducerWarps;  // keys of a tile that this warp copies
    const int row0 = (warp - Cfg::kProducerWarp) * kRows;
    constexpr int kPerKey = FP8 ? D / 16 : D / 8;      // 16-byte pieces of a key in the cache
    constexpr int kSteps = kRows * kPerKey / 32;
    constexpr int64_t kAbsent = -1, kUnknown = -2;     // no key; a page that the cache does not have
    const int es = FP8 ? 1 : 2;
    // lane l: key row0 + l
    auto entry_of = [&](const Walk<KEYS>& at, int t) {
      const int j = t * KEYS + row0 + lane;
      if (!at.more() || lane >= kRows || j >= at.s.len) return -1;
      return (int)ld_operand(a.page_table + (int64_t)at.b * a.page_table_ld + fast_div(j, p.page_div));
    };
    int64_t off[2];
    auto offsets = [&](const Walk<KEYS>& at, int t, int entry) {
      const int j = t * KEYS + row0 + lane;
      if (lane >= kRows || j >= at.s.len) {
        off[0] = off[1] = kAbsent;
      } else if (entry < 0 || entry >= a.pages) {
        off[0] = kUnknown;
        off[1] = kAbsent;
      } else {
        const int in_page = j - fast_div(j, p.page_div) * a.page_size;
        off[0] = (entry * a.k_page + in_page * a.k_token + at.h * a.k_head) * es;
        off[1] = (entry * a.v_page + in_page * a.v_token + at.h * a.v_head) * es;
      }
    };
    const uint32_t nan2 = 0x7fff7fffu;
    uint32_t it = 0;
    auto ready = [&](uint32_t stage) {  // this thread's part of the stage is in shared memory
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(full_bar(stage % S));
    };
    int t = w.t0, entry = entry_of(w, t);
    if constexpr (!FP8) {
      while (w.more() && ok) {
        offsets(w, t, entry);
        if (++t == w.t1) {
          w.next();
          t = w.t0;
        }
        entry = entry_of(w, t);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++it) {
          const int s = it % S;
          ok = ok && ptx::mbar_wait(empty_bar(s), ((it / S) & 1) ^ 1, abort_flag);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          const uint8_t* src = static_cast<const uint8_t*>(kv ? a.v_cache : a.k_cache);
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            const int piece = i * 32 + lane, r = piece / kPerKey, c = piece % kPerKey, row = row0 + r;
            const int64_t o = __shfl_sync(0xffffffffu, off[kv], r);
            const uint32_t dst = sKV + s * Cfg::kStage + (c >> 3) * (KEYS * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
            if (o == kUnknown) ptx::st_shared_16(dst, make_uint4(nan2, nan2, nan2, nan2));
            else ptx::cp_async_16(dst, src + (o < 0 ? 0 : o + c * 16), o < 0 ? 0u : 16u);
          }
          ptx::cp_async_commit();
          if (it >= Cfg::kAhead) {
            ptx::cp_async_wait<Cfg::kAhead>();
            ready(it - Cfg::kAhead);
          }
        }
      }
      ptx::cp_async_wait<0>();
      if (ok)
        for (uint32_t s = it > Cfg::kAhead ? it - Cfg::kAhead : 0; s < it; ++s) ready(s);
    } else {
      // Codes pass through registers: the pieces of kDepth stages are under way, the oldest is widened and stored
      constexpr int kDepth = 3;
      uint4 raw[kDepth][kSteps];
      const uint32_t total = 2 * (uint32_t)line[1];
      uint32_t asked = 0;
      auto request = [&](uint4 (&to)[kSteps]) {
        const int kv = asked & 1;
        if (asked >= total) return;
        if (kv == 0) {
          offsets(w, t, entry);
          if (++t == w.t1) {
            w.next();
            t = w.t0;
          }
          entry = entry_of(w, t);
        }
        ++asked;
        const uint8_t* src = static_cast<const uint8_t*>(kv ? a.v_cache : a.k_cache);
        const int64_t mine = kv ? off[1] : off[0];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const int piece = i * 32 + lane, r = piece / kPerKey, c = piece % kPerKey;
          const int64_t o = __shfl_sync(0xffffffffu, mine, r);
          const uint32_t fill = o == kUnknown ? 0x7f7f7f7fu : 0u;
          to[i] = make_uint4(fill, fill, fill, fill);
          if (o >= 0) to[i] = ld_stream_16(src + o + c * 16);
        }
      };
#pragma unroll
      for (int u = 0; u < kDepth; ++u) request(raw[u]);
      while (it < total && ok) {
#pragma unroll
        for (int u = 0; u < kDepth; ++u) {
          if (it >= total) break;
          const int s = it % S;
          ok = ok && ptx::mbar_wait(empty_bar(s), ((it / S) & 1) ^ 1, abort_flag);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int i = 0; i < kSteps; ++i) {
            const int piece = i * 32 + lane, r = piece / kPerKey, row = row0 + r;
            const uint32_t words[4] = {raw[u][i].x, raw[u][i].y, raw[u][i].z, raw[u][i].w};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int c = (piece % kPerKey) * 2 + half;
              uint32_t o[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) o[k] = widen2<T>((words[half * 2 + (k >> 1)] >> (16 * (k & 1))) & 0xffffu);
              ptx::st_shared_16(sKV + s * Cfg::kStage + (c >> 3) * (KEYS * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4),
                                make_uint4(o[0], o[1], o[2], o[3]));
            }
          }
          ready(it);
          ++it;
          request(raw[u]);
        }
      }
    }
    grid_launch_dependents();
  } else if (warp == Cfg::kQWarp) {
    // ------------------------------------------------------------------ query rows
    for (int seg = 0; w.more() && ok; w.next(), ++seg) {
      ok = ptx::mbar_wait(q_empty, (seg & 1) ^ 1, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      const int rows = min(128, w.s.n * p.group - w.qt * 128);
      constexpr int kPerRow = D / 8;
#pragma unroll 8
      for (int i = lane; i < rows * kPerRow; i += 32) {
        const int r = i / kPerRow, c = i % kPerRow, at = w.qt * 128 + r, token = fast_div(at, p.group_div);
        const T* src = static_cast<const T*>(a.q) + (int64_t)(w.s.start + token) * a.q_token + (w.h * p.group + at - token * p.group) * a.q_head;
        ptx::st_shared_16(sQ + (c >> 3) * (128 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4), ld_stream_16(src + c * 8));
      }
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(q_full);
    }
  } else if (warp == Cfg::kMmaWarp) {
    // ------------------------------------------------------------------ both products
    if (ptx::elect_one()) {
      constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
      constexpr uint32_t idesc_s = ptx::idesc_f16_f32(kBf16, false, 128, KEYS), idesc_o = ptx::idesc_f16_f32(kBf16, true, 128, D);
      uint32_t it = 0, g = 0;  // stages and tiles of this CTA so far
      // stages of the ring: keys of tile x in 2 x, its values in 2 x + 1
      auto scores = [&](uint32_t x, bool last) {
        const uint32_t st = it + 2 * x, s = st % S;
        if (!ptx::mbar_wait(full_bar(s), (st / S) & 1, abort_flag)) return false;
        ptx::tc_fence_after();
        const uint32_t d = tmem_base + ((g + x) & 1) * KEYS;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t at = (k & 3) * 32;
          ptx::mma_f16_ss(d, ptx::smem_desc_sw128(sQ + (k >> 2) * (128 * 128) + at),
                          ptx::smem_desc_sw128(sKV + s * Cfg::kStage + (k >> 2) * (KEYS * 128) + at), idesc_s, k > 0);
        }
        ptx::mma_commit(empty_bar(s));
        ptx::mma_commit(s_full((g + x) & 1));
        if (last) ptx::mma_commit(q_empty);
        return true;
      };
      auto output = [&](uint32_t x) {
        const uint32_t st = it + 2 * x + 1, s = st % S;
        if (!ptx::mbar_wait(full_bar(s), (st / S) & 1, abort_flag)) return false;
        if (!ptx::mbar_wait(p_full((g + x) & 1), ((g + x) >> 1) & 1, abort_flag)) return false;
        ptx::tc_fence_after();
        const uint32_t pt = tmem_base + ((g + x) & 1) * KEYS;
#pragma unroll
        for (int k = 0; k < KEYS / 16; ++k)
          ptx::mma_f16_ts(tmem_base + Cfg::kTmemO, pt + k * 8, ptx::smem_desc_mn_sw128(sKV + s * Cfg::kStage + k * 2048, KEYS * 128), idesc_o,
                          x > 0 || k > 0);
        ptx::mma_commit(empty_bar(s));
        ptx::mma_commit(o_done);
        return true;
      };
      for (int seg = 0; w.more() && ok; w.next(), ++seg) {
        const uint32_t n = w.t1 - w.t0;
        ok = ptx::mbar_wait(q_full, seg & 1, abort_flag);
        for (uint32_t x = 0; x < n && ok; ++x) {
          ok = scores(x, x + 1 == n);
          if (ok && x > 0) ok = output(x - 1);
        }
        ok = ok && output(n - 1);
        it += 2 * n;
        g += n;
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax: a thread per row
    const int r = threadIdx.x;
    SplitRows begun = {0, 0, 0, 0, 0};
    uint32_t g = 0;
    for (; w.more() && ok; w.next()) {
      const Seq& s = w.s;
      const int rows = min(128, s.n * p.group - w.qt * 128);
      const bool busy = (warp * 32) < rows;  // the same for the whole warp
      const int at = w.qt * 128 + min(r, rows - 1), token = fast_div(at, p.group_div), head = w.h * p.group + at - token * p.group;
      const int first_token = fast_div(w.qt * 128, p.group_div), prefix = s.len - s.n;
      float c = p.scale_log2;
      if (FP8 && a.k_scale) c *= ld_operand(a.k_scale + (a.k_scales > 1 ? w.h : 0));
      float m = -INFINITY, l = 0.f;  // reference of the exponents; sum
      for (int t = w.t0; t < w.t1; ++t, ++g) {
        ok = ptx::mbar_wait(s_full(g & 1), (g >> 1) & 1, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        if (busy) {
          ptx::tc_fence_after();
          const uint32_t ts = lane_base + (g & 1) * KEYS;
          uint32_t v[KEYS / 32][32];
#pragma unroll
          for (int k = 0; k < KEYS / 32; ++k) ptx::tmem_ld32(ts + k * 32, v[k]);
#pragma unroll
          for (int k = 0; k < KEYS / 32; ++k) ptx::tmem_ld_wait(v[k]);
          const int j0 = t * KEYS;
          // keys that every row of the tile sees need no mask
          if (j0 + KEYS > (a.mask ? prefix : prefix + first_token + 1)) {
#pragma unroll
            for (int k = 0; k < KEYS / 32; ++k) {
              const int j = j0 + k * 32, sees = (a.mask ? prefix : min(s.len, prefix + token + 1)) - j;  // keys seen of these 32
              uint32_t bits = sees >= 32 ? 0xffffffffu : sees <= 0 ? 0u : (1u << sees) - 1u;
              if (a.mask) {
                const volatile uint8_t* line_of_mask = static_cast<const uint8_t*>(a.mask) + (int64_t)(s.start + token) * a.mask_ld;
                const int end = min(min(32, s.len - j), a.mask_width + prefix - j);
                for (int i = max(sees, 0); i < end; ++i) bits |= (line_of_mask[j + i - prefix] ? 1u : 0u) << i;
              }
#pragma unroll
              for (int i = 0; i < 32; ++i) v[k][i] = (bits >> i) & 1u ? v[k][i] : 0xff800000u;
            }
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int k = 0; k < KEYS / 32; ++k)
#pragma unroll
            for (int i = 0; i < 32; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(v[k][i]));
          const float largest = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c;
          const bool move = largest > m + kSlack;
          const float m_new = move ? largest : m, factor = move ? ptx::ex2(m - m_new) : 1.f, minus_m = m_new == -INFINITY ? 0.f : -m_new;
          l *= factor;
          m = m_new;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < KEYS / 32; ++k) {
            uint32_t out[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float e0 = ptx::ex2(fmaf(__uint_as_float(v[k][2 * i]), c, minus_m)), e1 = ptx::ex2(fmaf(__uint_as_float(v[k][2 * i + 1]), c, minus_m));
              out[i] = pack2<T>(e0, e1);
              if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                // the weights as they are multiplied: a row that one key rules comes out as that key's value, without the rounding of its weight
                sum[i & 3] += __uint_as_float(out[i] << 16);
                sum[i & 3] += __uint_as_float(out[i] & 0xffff0000u);
              } else {
                sum[i & 3] += e0;
                sum[i & 3] += e1;
              }
            }
            ptx::tmem_st16(ts + k * 16, out);  // over scores that are in registers
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          // O of the tiles before this one is complete: waited for in every tile, so that the barrier is never two phases ahead
          if (g > 0) ok = ptx::mbar_wait(o_done, (g - 1) & 1, abort_flag);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          if (t > w.t0 && __any_sync(0xffffffffu, move)) {
            ptx::tc_fence_after();
#pragma unroll 1
            for (int d = 0; d < D; d += 16) {
              uint32_t o[32], n[16];
              ptx::tmem_ld16(lane_base + Cfg::kTmemO + d, o);
              ptx::tmem_ld_wait16(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) n[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
              ptx::tmem_st16(lane_base + Cfg::kTmemO + d, n);
            }
          }
          ptx::tmem_st_wait();
          ptx::tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(p_full(g & 1));
      }
      if (!ok) break;
      const bool whole = w.t0 == 0 && w.t1 == s.key_tiles;
      if (!whole && w.t0 == 0)
        begun = {s.start, w.qt, w.h, s.n * p.group, 1 + (int)((s.key_tiles - w.t1 + line[2] - 1) / line[2])};
      if (busy) {
        ok = ptx::mbar_wait(o_done, (g - 1) & 1, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        if (whole) {
          const float inv = l == 0.f ? 0.f : (FP8 && a.v_scale ? ld_operand(a.v_scale + (a.v_scales > 1 ? w.h : 0)) : 1.f) / l;
          T* dst = static_cast<T*>(a.out) + ((int64_t)(s.start + token) * a.q_heads + head) * D;
#pragma unroll 1
          for (int d = 0; d < D; d += 16) {
            uint32_t o[32], n[8];
            ptx::tmem_ld16(lane_base + Cfg::kTmemO + d, o);
            ptx::tmem_ld_wait16(o);
            // a row that sees nothing is zero, whatever its weights of zero met
#pragma unroll
            for (int i = 0; i < 8; ++i)
              n[i] = l == 0.f ? 0u : pack2<T>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
            if (r < rows) {
              reinterpret_cast<uint4*>(dst + d)[0] = make_uint4(n[0], n[1], n[2], n[3]);
              reinterpret_cast<uint4*>(dst + d)[1] = make_uint4(n[4], n[5], n[6], n[7]);
            }
          }
          if (a.lse && r < rows) a.lse[(int64_t)(s.start + token) * a.q_heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        } else {
          const int64_t slot = (2 * (int64_t)blockIdx.x + (w.t0 == 0 ? 1 : 0)) * p.row_slots + r;
          float* dst = p.part_o + slot * D;
#pragma unroll 1
          for (int d = 0; d < D; d += 16) {
            uint32_t o[32];
            ptx::tmem_ld16(lane_base + Cfg::kTmemO + d, o);
            ptx::tmem_ld_wait16(o);
            if (r < rows)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                reinterpret_cast<uint4*>(dst + d)[i] = l == 0.f ? make_uint4(0, 0, 0, 0) : make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
          if (r < rows) p.part_ml[slot] = make_float2(m, l);
        }
        ptx::tc_fence_before();
      }
    }
    if (threadIdx.x == 0) p.split[blockIdx.x] = begun;
  }

  if (*abort_flag) {  // a wait gave up: products that are still under way end before the shared memory goes
    const unsigned long long t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) atomicCAS(p.status, 0, 1);
  if (warp == Cfg::kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, 512);
  }
}

// Rows whose keys were cut: a warp per row adds up its pieces, in the order of the line.
template <typename T, int D, bool FP8>
__global__ void __launch_bounds__(256) tree_attention_join_kernel(const __grid_constant__ AttnParams p) {
  const b200_tree_attention_args& a = p.a;
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, cta = blockIdx.x, r = blockIdx.y * 8 + (threadIdx.x >> 5);
  const volatile int* const from = reinterpret_cast<const volatile int*>(p.split + cta);
  const int parts = from[4];
  if (parts == 0) return;
  const int start = from[0], qt = from[1], h = from[2], row = qt * 128 + r;
  if (r >= 128 || row >= from[3]) return;
  auto slot_of = [&](int i) { return (2 * (int64_t)(cta + i) + (i == 0 ? 1 : 0)) * p.row_slots + r; };
  auto ml_of = [&](int i) {
    const volatile float* ml = reinterpret_cast<const volatile float*>(p.part_ml + slot_of(i));
    return make_float2(ml[0], ml[1]);
  };
  float m = -INFINITY;
  for (int i = lane; i < parts; i += 32) m = fmaxf(m, ml_of(i).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float ref = m == -INFINITY ? 0.f : m;
  constexpr int kPer = D / 32;
  float sum = 0.f, acc[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
  for (int i0 = 0; i0 < parts; i0 += 32) {
    float weight = 0.f;
    if (i0 + lane < parts) {
      const float2 ml = ml_of(i0 + lane);
      weight = ptx::ex2(ml.x - ref);
      sum = fmaf(ml.y, weight, sum);
    }
    const int n = min(32, parts - i0);
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float f = __shfl_sync(0xffffffffu, weight, i);
      const volatile float* src = p.part_o + slot_of(i0 + i) * D + lane * kPer;
#pragma unroll
      for (int k = 0; k < kPer; ++k) acc[k] = fmaf(src[k], f, acc[k]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int token = fast_div(row, p.group_div), head = h * p.group + row - token * p.group;
  const int64_t to = (int64_t)(start + token) * a.q_heads + head;
  const float inv = sum == 0.f ? 0.f : (FP8 && a.v_scale ? ld_operand(a.v_scale + (a.v_scales > 1 ? h : 0)) : 1.f) / sum;
  T* dst = static_cast<T*>(a.out) + to * D + lane * kPer;
#pragma unroll
  for (int k = 0; k < kPer; ++k) dst[k] = from_f32<T>(acc[k] * inv);
  if (a.lse && lane == 0) a.lse[to] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
}

// CTAs of a call: no more than there can be tiles
inline int64_t attention_grid(const b200_tree_attention_args& a) {
  const int keys = a.dim > 128 ? 64 : 128;
  const int64_t group = a.q_heads / a.kv_heads, row_tiles = cdiv(a.tokens * group, 128) + a.sequences;
  const int64_t capacity = a.max_pages * a.page_size, key_tiles = capacity > 0 ? cdiv(capacity, keys) : 1;
  const double tiles = (double)row_tiles * a.kv_heads * key_tiles;
  const int sms = sm_count();
  return tiles < sms ? (int64_t)tiles : sms;
}
inline int attention_row_slots(const b200_tree_attention_args& a) {
  const int64_t rows = a.tokens * (a.q_heads / a.kv_heads);
  return rows < 128 ? (int)rows : 128;
}
struct AttnWorkspace {
  size_t ml, split, total;  // byte offsets behind the partial sums
};
inline AttnWorkspace attention_workspace(const b200_tree_attention_args& a) {
  const int64_t grid = attention_grid(a), slots = 2 * grid * attention_row_slots(a);
  AttnWorkspace w;
  w.ml = align_up((size_t)slots * a.dim * 4, 256);
  w.split = align_up(w.ml + (size_t)slots * 8, 256);
  w.total = w.split + (size_t)grid * sizeof(SplitRows);
  return w;
}

template <typename T, int D, bool FP8>
static int launch_attention(const AttnParams& p, int grid, cudaStream_t st) {
  using Cfg = AttnCfg<D, FP8>;
  auto k = tree_attention_kernel<T, D, FP8>;
  if (int rc = allow_smem(k, Cfg::kSmemBytes, "tree_attention_kernel")) return rc;
  if (int rc = launch_dependent(k, dim3((unsigned)grid), Cfg::kThreads, Cfg::kSmemBytes, st, 1, "tree_attention", p)) return rc;
  return launch_dependent(tree_attention_join_kernel<T, D, FP8>, dim3((unsigned)grid, (unsigned)cdiv(p.row_slots, 8)), 256, 0, st, 1,
                          "tree_attention", p);
}
template <typename T, int D>
static int launch_attention(const AttnParams& p, int grid, cudaStream_t st) {
  return p.a.cache_dtype == B200_E4M3 ? launch_attention<T, D, true>(p, grid, st) : launch_attention<T, D, false>(p, grid, st);
}
template <typename T>
static int launch_attention(const AttnParams& p, int grid, cudaStream_t st) {
  switch (p.a.dim) {
    case 64: return launch_attention<T, 64>(p, grid, st);
    case 128: return launch_attention<T, 128>(p, grid, st);
    default: return launch_attention<T, 256>(p, grid, st);
  }
}

static int check_attention(const b200_tree_attention_args& a) {
  B200_CHECK_ARG(a.tokens >= 0 && a.sequences >= 0 && a.q_heads > 0 && a.kv_heads > 0 && a.q_heads % a.kv_heads == 0,
                 "tree_attention: %d query heads over %d kv heads", a.q_heads, a.kv_heads);
  B200_CHECK_ARG(a.dtype == B200_BF16 || a.dtype == B200_F16, "tree_attention: unknown dtype code %d", a.dtype);
  B200_CHECK_ARG(a.cache_dtype == a.dtype || a.cache_dtype == B200_E4M3, "tree_attention: the cache has the queries' type or E4M3");
  B200_UNSUPPORTED(a.dim != 64 && a.dim != 128 && a.dim != 256, "tree_attention: heads of %d (64, 128 and 256 are built)", a.dim);
  B200_CHECK_ARG(a.page_size > 0 && a.pages >= 0 && a.max_pages >= 0, "tree_attention: pages");
  B200_UNSUPPORTED(a.tokens * (int64_t)a.q_heads > 0x3fffffffLL || a.sequences > 0x3fffffffLL || a.max_pages > 0x7fffffffLL ||
                       a.pages > 0x7fffffffLL || a.max_pages * a.page_size > 0x7fffff00LL,
                   "tree_attention: more than 2^30 query rows or sequences, or a page table of more than 2^31 tokens a line");
  B200_CHECK_ARG(a.scale > 0.f, "tree_attention: the scale is positive");
  return B200_OK;
}

}  // namespace b200

extern "C" size_t b200_tree_attention_workspace_bytes(const b200_tree_attention_args* args) {
  using namespace b200;
  if (!args || check_attention(*args) != B200_OK || args->tokens == 0 || args->sequences == 0) return 0;
  return attention_workspace(*args).total;
}

extern "C" int b200_tree_attention(const b200_tree_attention_args* args, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace b200;
  B200_CHECK_ARG(args != nullptr, "tree_attention: null pointer");
  AttnParams p = {};
  p.a = *args;
  const b200_tree_attention_args& a = p.a;
  if (int rc = check_attention(a)) return rc;
  if (a.tokens == 0 || a.sequences == 0) return B200_OK;
  B200_CHECK_ARG(a.q && a.out && a.seq_lens && (a.max_pages == 0 || (a.page_table && (a.pages == 0 || (a.k_cache && a.v_cache)))),
                 "tree_attention: null pointer");
  const int per16 = a.cache_dtype == B200_E4M3 ? 16 : 8;  // elements of 16 bytes
  B200_CHECK_ARG(((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)a.k_cache | (uintptr_t)a.v_cache) % 16 == 0 && (a.q_token | a.q_head) % 8 == 0 &&
                     (a.k_page | a.k_token | a.k_head | a.v_page | a.v_token | a.v_head) % per16 == 0,
                 "tree_attention: heads of q and of the caches start at multiples of 16 bytes");
  B200_CHECK_ARG(((uintptr_t)a.page_table | (uintptr_t)a.seq_lens | (uintptr_t)a.q_starts | (uintptr_t)a.lse) % 4 == 0, "tree_attention: misaligned pointer");
  B200_CHECK_ARG((!a.k_scale && !a.v_scale) || a.cache_dtype == B200_E4M3, "tree_attention: scales belong to an E4M3 cache");
  B200_CHECK_ARG((!a.k_scale || a.k_scales == 1 || a.k_scales == a.kv_heads) && (!a.v_scale || a.v_scales == 1 || a.v_scales == a.kv_heads),
                 "tree_attention: one scale, or one per kv head");
  B200_CHECK_ARG(!a.mask || a.mask_width >= 0, "tree_attention: mask width");
  const AttnWorkspace ws = attention_workspace(a);
  if (!workspace || workspace_bytes < ws.total || (uintptr_t)workspace % 16) {
    set_error_detail("tree_attention: workspace of %zu bytes, %zu needed, 16-byte aligned", workspace_bytes, ws.total);
    return B200_E_WORKSPACE;
  }
  p.group = a.q_heads / a.kv_heads;
  p.group_div = make_fastdiv(p.group);
  p.page_div = make_fastdiv(a.page_size);
  p.row_slots = attention_row_slots(a);
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.capacity = a.max_pages * a.page_size;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + ws.ml);
  p.split = reinterpret_cast<SplitRows*>(static_cast<uint8_t*>(workspace) + ws.split);
  p.status = device_status_word();
  if (!p.status) {
    set_error_detail("cannot resolve the device status word");
    return B200_E_LAUNCH;
  }
  const int grid = (int)attention_grid(a);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a.dtype == B200_BF16 ? launch_attention<__nv_bfloat16>(p, grid, st) : launch_attention<__half>(p, grid, st);
}
