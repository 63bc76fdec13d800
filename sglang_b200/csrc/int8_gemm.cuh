// Product of 8-bit integers with a scale per token and per output channel:
//     C[m, n] = (sum_k A[m, k] * B[n, k]) * sa[m] * sb[n] (+ bias[n])
// tcgen05.mma kind::i8 adds up in 32-bit integers, exactly, so the sum stays in TMEM for all of K, the order of the additions does
// not matter, and one pass over it at the end applies both scales: three roundings in fp32 and the last one to the output type.
#pragma once

#include "gemm_pair.cuh"
#include "int8_round.cuh"

namespace b200 {

namespace ptx {
__device__ __forceinline__ void mma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
      "}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void st_cluster_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// 16 bytes to another CTA's shared memory, counted on a barrier there: whoever waits for the bytes sees them, without a barrier of
// the whole cluster (0.75 us with the release of everything written before it)
__device__ __forceinline__ void st_async_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr), "r"(a),
               "r"(b), "r"(c), "r"(d), "r"(bar)
               : "memory");
}
// As mbar_wait, for bytes that another CTA of the cluster wrote
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  const unsigned long long t0 = globaltimer_ns();
  for (uint32_t spin = 1;; ++spin) {
    uint32_t ok;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((spin & 63u) == 0u) {
      if (*abort_flag) return false;
      if (globaltimer_ns() - t0 > kWaitLimitNs) {
        *abort_flag = 1;
        return false;
      }
    }
  }
}
// Cluster barrier that orders nothing but the CTAs' progress: 0.35 us, with release and acquire 0.75
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ int4 ld_shared_i4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
// Instruction descriptor for kind::i8, signed x signed -> int32 (no saturation), both operands K-major.
//   bits 4-5 D format (2 = s32)  7-9 A format (1 = signed)  10-12 B format  17-22 N >> 3  24-28 M >> 4
__host__ __device__ constexpr uint32_t idesc_s8_s32(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
}  // namespace ptx

struct Int8Params {
  const float *sa, *sb;  // [M], [N]
  const void* x;         // QUANT: 16-bit rows [M, K], x_ld elements apart
  int64_t x_ld;
  const void* bias;      // [N] of the output's type, or null
  void* C;               // [M, N], contiguous
  const int8_t* w;       // B, for prefetches
  int64_t w_ld;
  int M, N, K, num_kb;
  int n_tiles, t_tiles;
  int nt, k_splits, kb_per_split;           // stream kernel: tokens of a tile, K splits of an item (one cluster)
  int m_tiles, group_m;                     // pair kernel
  FastDiv per_group_div;
  int* status;
};

// Few tokens. The roles of the operands are swapped: 128 rows of B fill the lanes of the tensor-core tile, nt tokens (a multiple of
// 16, at most NT) are its columns, so that few tokens waste little and a thread of the epilogue owns one output channel.
// Work item = (128 rows of B, nt tokens, K split); one CTA each. The K splits of an item are one cluster: they exchange their integer
// sums through distributed shared memory, every one of them adding up and storing its share of the tokens.
// Sums of four tokens travel as one 16-byte store per lane: 203 x 4096 x 14336 in four splits 25.3 us a word at a time, 22.9 so.
constexpr int kInt8MaxSplits = 8;
__host__ __device__ constexpr int int8_share(int rows, int splits) { return ((rows + splits - 1) / splits + 3) / 4 * 4; }  // tokens per split
constexpr int int8_sum_rows(int nt) {
  int most = 0;
  for (int s = 2; s <= kInt8MaxSplits; ++s) most = s * int8_share(nt, s) > most ? s * int8_share(nt, s) : most;
  return most;
}

template <int NT, bool QUANT>
struct Int8StreamCfg {
  static constexpr int kStageW = 128 * kBK, kStageX = NT * kBK;
  static constexpr int kCtasPerSm = NT <= 64 ? 2 : 1;
  static constexpr int kStages = NT == 16 ? 5 : NT == 32 ? 4 : NT == 64 ? 4 : NT == 128 ? 6 : 4;
  // With many tokens two epilogue warps share 32 channels and take every second 16 tokens each
  static constexpr int kEpiWarps = NT <= 32 ? 4 : 8, kEpiThreads = kEpiWarps * 32;
  static constexpr int kProducerWarp = kEpiWarps, kMmaWarp = kEpiWarps + 1;
  static constexpr int kQuantRows = 4, kQuantWarps = 4;  // QUANT: rows that the quantiser warps cover
  static constexpr int kThreads = kEpiThreads + 64 + (QUANT ? kQuantWarps * 32 : 0);
  static constexpr int kTmemCols = NT < 32 ? 32 : NT;
  // sums of the splits, [split][tokens of this CTA / 4][128][4]; with many tokens they go to the ring once it is idle
  static constexpr int kSumBytes = NT <= 32 ? int8_sum_rows(NT) * 512 : 0;
  static constexpr size_t kSmemBytes = (size_t)kStages * (kStageW + kStageX) + kSumBytes + NT * 4 + (QUANT ? 32 : 0) + 1024 + 256;
  // Few sums travel as stores that count themselves (1 x 6144 x 4096 in four splits 7.7 -> 7.1 us), many as plain ones with one barrier
  // behind them, which are faster by the byte (203 x 4096 x 14336 22.4 against 19.9)
  static constexpr bool kCounted = NT <= 64;
  static_assert(kSumBytes > 0 || int8_sum_rows(NT) * 512 <= kStages * (kStageW + kStageX), "the sums fit the ring");
};

// QUANT: A is the 16-bit input of a linear layer, up to four rows. While the weights fill the ring, every CTA finds the rows' largest
// magnitudes (the epilogue warps and four more, a whole row from L2), then the four quantise the K blocks of the CTA into the ring,
// bit for bit as the stand-alone quantiser does: one launch for the layer instead of two.
template <int NT, bool QUANT, typename OutT>
__global__ void __launch_bounds__(Int8StreamCfg<NT, QUANT>::kThreads)
int8_stream_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const Int8Params p) {
  using Cfg = Int8StreamCfg<NT, QUANT>;
  constexpr int S = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_al = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
  const uint32_t sW = smem_base, sX = smem_base + S * Cfg::kStageW;
  constexpr uint32_t kRing = S * (Cfg::kStageW + Cfg::kStageX), kSums = Cfg::kSumBytes ? kRing : 0;
  float* sa = reinterpret_cast<float*>(smem_al + kRing + Cfg::kSumBytes);  // [NT]
  float* tops = sa + NT;                                                   // QUANT: [rows][parts of a row], one a warp
  uint64_t* bars = reinterpret_cast<uint64_t*>(tops + (QUANT ? 8 : 0));
  const uint32_t bar0 = ptx::smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (S + s); };
  const uint32_t done_bar = bar0 + 8u * 2 * S, sum_bar = done_bar + 8u;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(bars + 2 * S + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * S + 3);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kProducerWarp = Cfg::kProducerWarp, kMmaWarp = Cfg::kMmaWarp;
  const int splits = p.k_splits, tile = blockIdx.x / splits, ks = blockIdx.x - tile * splits;
  const int n_tile = tile / p.t_tiles, n0 = n_tile * 128, m0 = (tile - n_tile * p.t_tiles) * p.nt;
  const int kb0 = ks * p.kb_per_split, kb1 = min(p.num_kb, kb0 + p.kb_per_split);
  const int rows = min(p.nt, p.M - m0);
  // K splits: token t belongs to split t / share, this one's are t0 .. t0 + mine
  const int share = int8_share(rows, splits), groups = share / 4, t0 = ks * share, mine = min(share, rows - t0);
  // QUANT: 16 groups of eight lanes take four rows of four K blocks side by side. Four K blocks are fewer than the ring's stages: with more
  // under way a group would wait for a phase of a stage's barrier that is two ahead of it, which the parity does not tell
  // from the one before.
  constexpr int kQuantRows = Cfg::kQuantRows;
  static_assert(!QUANT || (NT == 16 && S > 4), "the K blocks under way fit the ring");

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      ptx::mbar_init(full_bar(s), QUANT ? 1 + kQuantRows : 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    ptx::mbar_init(done_bar, 1);
    ptx::mbar_init(sum_bar, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    // sums of every split for this CTA's tokens, four tokens of 128 channels at a time
    if (Cfg::kCounted && splits > 1) ptx::mbar_expect_tx(sum_bar, (uint32_t)(splits * ((max(mine, 0) + 3) / 4) * 2048));
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), Cfg::kTmemCols);
    ptx::tmem_relinquish();
  }
  if (warp == kProducerWarp && lane == 0) {
    ptx::prefetch_tensormap(&tmap_w);
    if (!QUANT) ptx::prefetch_tensormap(&tmap_x);
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // "I have started, my barriers are initialised", waited for before another CTA's shared memory is written at the very end
  if (splits > 1) ptx::cluster_arrive_relaxed();
  // This grid is launched as a programmatic dependent: every operand, and at the end the output, belongs to the kernels before it
  // in the stream, which may still run. Until then the weights are only asked for, as a prefetch into L2, a row each.
  if (warp < 4 && n0 + (int)threadIdx.x < p.N)
    prefetch_weight_row(reinterpret_cast<const uint8_t*>(p.w) + (int64_t)(n0 + threadIdx.x) * p.w_ld + kb0 * kBK, min(kPrefetchKb, kb1 - kb0));
  const int64_t zero = grid_dependency_zero();

  bool ok = true;
  float sb = 0.f, bias = 0.f, scale_of_lane = 0.f;
  const int r = threadIdx.x & 127, half = warp >> 2, n = n0 + r;  // of an epilogue thread
  constexpr int kNext = Cfg::kEpiWarps * 4;                       // tokens until its next 16
  const uint32_t lane_base = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
  OutT* const out = static_cast<OutT*>(p.C) + (int64_t)m0 * p.N + n;
  // Four tokens of this thread's channel. The values come first and the stores are all that a predicate guards: with a branch around
  // each token's arithmetic the epilogue of 256 tokens took 10 us.
  auto store4 = [&](int t, int a, int b, int c, int d) {
    const float4 s4 = ld_shared_f4(sa + t);
    const OutT o[4] = {from_f32<OutT>(fmaf((float)a * s4.x, sb, bias)), from_f32<OutT>(fmaf((float)b * s4.y, sb, bias)),
                       from_f32<OutT>(fmaf((float)c * s4.z, sb, bias)), from_f32<OutT>(fmaf((float)d * s4.w, sb, bias))};
    const int here = n < p.N ? rows - t : 0;
    OutT* to = out + (int64_t)t * p.N;
#pragma unroll
    for (int i = 0; i < 4; ++i, to += p.N)
      if (i < here) *to = o[i];
  };
  // QUANT: eight lanes hold the 128 values of one (row, K block), 16 each; the groups of a warp have the same K block
  constexpr int kStep = 4 * Cfg::kQuantWarps / kQuantRows, kAhead = 4;  // K blocks side by side, and in flight per group
  const int q_tid = threadIdx.x - (kMmaWarp + 1) * 32, chunk = q_tid & 7, q_row = (q_tid >> 3) & (kQuantRows - 1);
  const int first = (q_tid >> 3) / kQuantRows, nkb = kb1 - kb0;
  uint4 raw[kAhead][2];
  auto request = [&](int j, int u) {
    const int k = (kb0 + j) * kBK + chunk * 16;  // K is a multiple of 16
    const OutT* src = static_cast<const OutT*>(p.x) + (m0 + min(q_row, rows - 1)) * p.x_ld + k + zero;
    const bool inside = j < nkb && k < p.K;
    raw[u][0] = inside ? ld_stream_16(src) : make_uint4(0, 0, 0, 0);
    raw[u][1] = inside ? ld_stream_16(src + 8) : make_uint4(0, 0, 0, 0);
  };
  if constexpr (QUANT) {
    if (warp > kMmaWarp)
#pragma unroll
      for (int u = 0; u < kAhead; ++u) request(first + u * kStep, u);
    // largest magnitudes: the eight warps that do not drive the pipeline share the rows evenly, 16 bytes a lane
    if (warp < kProducerWarp || warp > kMmaWarp) {
      const int w = warp < kProducerWarp ? warp : warp - 2;
      const int per_row = rows <= 1 ? 8 : rows <= 2 ? 4 : 2, row = w / per_row, part = w - row * per_row;
      float top = 0.f;
      if (row < rows) {
        const OutT* x = static_cast<const OutT*>(p.x) + (m0 + row) * p.x_ld + zero;
        const int nvec = p.K >> 3, step = per_row * 32;
        for (int i = part * 32 + lane; i < nvec; i += 8 * step) {
          uint4 part8[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) part8[u] = i + u * step < nvec ? ld_stream_16(x + (i + u * step) * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max_nan(top, fabsf(to_f32<OutT>(reinterpret_cast<const OutT*>(part8 + u)[e])));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
      }
      if (lane == 0) tops[w] = top;
      asm volatile("bar.sync 2, 256;" ::: "memory");
      // every warp on its own: no second barrier before the scales are used
      if (lane < kQuantRows) {
        float m = 0.f;
        for (int i = 0; i < per_row && lane < rows; ++i) m = max_nan(m, tops[lane * per_row + i]);
        scale_of_lane = int8_scale(m);
      }
      if (warp == 0 && lane < NT) sa[lane] = lane < rows ? scale_of_lane : 0.f;
    }
  }

  if (warp == kProducerWarp) {
    if (ptx::elect_one()) {
      const uint32_t bytes = Cfg::kStageW + (QUANT ? 0 : p.nt * kBK);
      uint32_t it = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int s = it % S;
        if (!ptx::mbar_wait(empty_bar(s), ((it / S) & 1) ^ 1, abort_flag)) break;
        ptx::mbar_expect_tx(full_bar(s), bytes);
        ptx::tma_load_2d(sW + s * Cfg::kStageW, &tmap_w, kb * kBK, n0, full_bar(s));
        if (!QUANT) ptx::tma_load_2d(sX + s * Cfg::kStageX, &tmap_x, kb * kBK, m0, full_bar(s));
      }
      // All that this CTA reads is on its way: what comes next may start. 1 x 4096 x 4096, 14336 5.0, 11.7 us; from the kernel's
      // start 5.4, 12.4 (its CTAs crowd this one's), with the sums complete 5.6, 12.7
      grid_launch_dependents();
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    if (ptx::elect_one()) {
      const uint32_t idesc = ptx::idesc_s8_s32(128, p.nt);
      uint32_t it = 0;
      for (int kb = kb0; kb < kb1 && ok; ++kb, ++it) {
        const int s = it % S;
        ok = ptx::mbar_wait(full_bar(s), (it / S) & 1, abort_flag);
        if (!ok) break;
        ptx::tc_fence_after();
        const uint64_t dw = ptx::smem_desc_sw128(sW + s * Cfg::kStageW), dx = ptx::smem_desc_sw128(sX + s * Cfg::kStageX);
#pragma unroll
        for (int k = 0; k < kBK / 32; ++k) ptx::mma_i8(tmem_base, dw + 2 * k, dx + 2 * k, idesc, it > 0 || k > 0);
        ptx::mma_commit(empty_bar(s));
      }
      if (ok) ptx::mma_commit(done_bar);
    }
    __syncwarp();
  } else if (QUANT && warp > kMmaWarp) {
    if constexpr (QUANT) {
      const unsigned group = 0xffu << (lane & 24);
      const float scale = __shfl_sync(0xffffffffu, scale_of_lane, min(q_row, rows - 1)), inv = __frcp_rn(scale);
      for (int j0 = 0; j0 < nkb; j0 += kAhead * kStep) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (j0 + u * kStep >= nkb) break;  // the same for the whole warp
          const int j = j0 + u * kStep + first;
          uint32_t c[2][8];
#pragma unroll
          for (int e = 0; e < 16; ++e)
            c[e >> 3][e & 7] = rint_bits(div_by(to_f32<OutT>(reinterpret_cast<const OutT*>(raw[u])[e]), scale, inv));
          const uint2 lo = pack8_s8(c[0]), hi = pack8_s8(c[1]);
          request(j + kAhead * kStep, u);
          if (j >= nkb) continue;
          const int s = j % S;
          ok = ok && ptx::mbar_wait(empty_bar(s), ((j / S) & 1) ^ 1, abort_flag);
          if (ok && q_row < rows) {
            const uint32_t dst = sX + s * Cfg::kStageX + q_row * 128 + ((chunk ^ q_row) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(lo.x), "r"(lo.y), "r"(hi.x), "r"(hi.y) : "memory");
            ptx::fence_proxy_async_smem();  // generic-proxy writes -> the tensor core's reads
          }
          __syncwarp(group);
          if (ok && chunk == 0) ptx::mbar_arrive(full_bar(s));
        }
      }
    }
    __syncwarp();
  } else {
    for (int t = threadIdx.x; !QUANT && t < NT; t += Cfg::kEpiThreads) sa[t] = t < rows ? ld_operand(p.sa + m0 + t) : 0.f;
    if (n < p.N) {
      sb = ld_operand(p.sb + n);
      if (p.bias != nullptr) bias = to_f32<OutT>(static_cast<const OutT*>(p.bias)[n]);
    }
    asm volatile("bar.sync 1, %0;" ::"n"(Cfg::kEpiThreads) : "memory");
    ok = ptx::mbar_wait(done_bar, 0, abort_flag);
    ptx::tc_fence_after();
    if (splits == 1 && ok) {
#pragma unroll 1
      for (int c = half * 16; c < rows; c += kNext) {
        uint32_t v[32];
        ptx::tmem_ld16(lane_base + c, v);
        ptx::tmem_ld_wait16(v);
#pragma unroll
        for (int t = 0; t < 16; t += 4) store4(c + t, (int)v[t], (int)v[t + 1], (int)v[t + 2], (int)v[t + 3]);
      }
    }
  }

  if (splits > 1) {
    __syncwarp();
    ptx::cluster_wait();
    if (Cfg::kSumBytes == 0) {  // every ring is idle: done_bar completes behind the last product
      ptx::cluster_arrive_relaxed();
      ptx::cluster_wait();
    }
    if (warp < Cfg::kEpiWarps) {
#pragma unroll 1
      for (int c = half * 16; c < rows; c += kNext) {
        uint32_t v[32];
        ptx::tmem_ld16(lane_base + c, v);
        int owner = c / share, g = (c - owner * share) / 4;
        ptx::tmem_ld_wait16(v);
#pragma unroll
        for (int t = 0; t < 16; t += 4) {
          const int cta = min(owner, splits - 1);
          const uint32_t to = ptx::mapa(smem_base + kSums + ((ks * groups + g) * 128 + r) * 16, cta);
          if (c + t < rows) {
            if (Cfg::kCounted) ptx::st_async_v4(to, v[t], v[t + 1], v[t + 2], v[t + 3], ptx::mapa(sum_bar, cta));
            else ptx::st_cluster_v4(to, v[t], v[t + 1], v[t + 2], v[t + 3]);
          }
          if (++g == groups) g = 0, ++owner;
        }
      }
    }
    __syncwarp();
    // "I have sent everything": counted sums are waited for by their bytes, and for this only before the CTA leaves
    if (Cfg::kCounted) ptx::cluster_arrive_relaxed();
    else ptx::cluster_sync();
    if (warp < Cfg::kEpiWarps) {
      if (ok && mine > 0 && (!Cfg::kCounted || ptx::mbar_wait_cluster(sum_bar, 0, abort_flag))) {
        const uint32_t src = smem_base + kSums + r * 16;
#pragma unroll 2
        for (int g = half; 4 * g < mine; g += Cfg::kEpiWarps / 4) {
          int4 sum = ptx::ld_shared_i4(src + g * 2048);
#pragma unroll 3
          for (int c = 1; c < splits; ++c) {
            const int4 v = ptx::ld_shared_i4(src + (c * groups + g) * 2048);
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
          }
          store4(t0 + 4 * g, sum.x, sum.y, sum.z, sum.w);
        }
      }
    }
    __syncwarp();
    if (Cfg::kCounted) ptx::cluster_wait();
  }

  if (*abort_flag) {  // a wait gave up: copies that are still under way land before the shared memory goes
    const unsigned long long t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) atomicCAS(p.status, 0, 1);
  if (warp == kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

// Row-major [rows, cols] matrix of `es`-byte elements, `ld` elements between rows, box [box_rows x box_cols] with the swizzle that fits
// its width. Encoded for every call.
inline int encode_tmap(CUtensorMap* m, CUtensorMapDataType type, int es, const void* base, int64_t rows, int64_t cols, int64_t ld,
                       int box_rows, int box_cols, CUtensorMapL2promotion promotion, const char* what) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) {
    set_error_detail("cuTensorMapEncodeTiled is not available from the driver");
    return B200_E_LAUNCH;
  }
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(ld * es)};
  cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  const int w = box_cols * es;
  CUresult r = enc(m, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   w == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                   : w == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                             : CU_TENSOR_MAP_SWIZZLE_NONE,
                   promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error_detail("cuTensorMapEncodeTiled(%s: rows=%lld cols=%lld ld=%lld box=%dx%d) failed with CUresult %d", what, (long long)rows,
                     (long long)cols, (long long)ld, box_rows, box_cols, (int)r);
    return B200_E_LAUNCH;
  }
  return B200_OK;
}
inline int encode_tmap_s8(CUtensorMap* m, const void* base, int64_t rows, int64_t k, int64_t ld, int box_rows, const char* what) {
  return encode_tmap(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, base, rows, k, ld, box_rows, kBK, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, what);
}

// p.nt tokens per tile (at most NT), p.k_splits splits. QUANT: p.x is quantised, A is null.
template <int NT, bool QUANT, typename OutT>
inline int launch_int8_stream(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t K, Int8Params p, cudaStream_t st) {
  using Cfg = Int8StreamCfg<NT, QUANT>;
  p.n_tiles = (int)cdiv(p.N, 128);
  p.t_tiles = (int)cdiv(p.M, p.nt);
  p.kb_per_split = (int)cdiv(p.num_kb, p.k_splits);
  p.K = (int)K;
  CUtensorMap tw, tx;
  if (int rc = encode_tmap_s8(&tw, B, p.N, K, ldb, 128, "B")) return rc;
  if (QUANT) tx = tw;
  else if (int rc = encode_tmap_s8(&tx, A, p.M, K, lda, p.nt, "A")) return rc;
  auto k = int8_stream_kernel<NT, QUANT, OutT>;
  if (int rc = allow_smem(k, Cfg::kSmemBytes, "int8_stream_kernel")) return rc;
  return launch_dependent(k, dim3((unsigned)(p.n_tiles * p.t_tiles * p.k_splits)), Cfg::kThreads, Cfg::kSmemBytes, st, (unsigned)p.k_splits,
                          "int8_stream_kernel", tw, tx, p);
}

}  // namespace b200
