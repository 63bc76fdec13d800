// Many tokens (see int8_gemm.cuh): persistent CTA pairs (tcgen05 cta_group::2), a tile of 256 rows and up to BN columns per pair.
// Each CTA loads its own 128 rows of A and half of the B tile: with 256 columns 32 KB per 128 of K, which at 128 B/clk in and
// out of shared memory fit the 512 clocks of its products. Two accumulators of BN columns in TMEM, so that the epilogue of a tile
// runs under the products of the next. The width of a tile is any multiple of 32: the launch takes the one that fills its waves.
// SWAP: the 256 rows are rows of B, output channels, and the columns are tokens, so that a tile's width divides their number evenly:
// 1027 tokens are multiplied as 5 x 224 and not as 5 x 256. A thread then owns a channel and its boxes are written by columns.
// Few tiles: the K splits of a tile, 2 or 4, are one cluster; every one of them sums and stores its share of the 32-column chunks,
// the others hand theirs over through distributed shared memory, into the ring, which is idle by then.
// Roles per CTA (320 threads):
//   warps 0-7  epilogue: warp w owns TMEM lanes 32 (w % 4).. and every second chunk of 32 columns; 32 x 32 boxes leave through bulk
//              tensor stores
//   warp  8    TMA producer (no multicast)      warp 9  MMA issuer (leader CTA only)
// Protocol of a pair (rank 0 = leader):
//   full[s]   (leader's)  2 arrivals (one expect_tx per producer) + the bytes of both CTAs' loads
//   empty[s]  (each CTA)  arrival from the leader's commit       tfull[b] (each CTA)  likewise, when a tile's sums are complete
//   tempty[b] (leader's)  16 arrivals: the epilogue warps of both CTAs, where a later tile of the pair uses the accumulator
#pragma once

#include "int8_gemm.cuh"

namespace b200 {

namespace ptx {
__device__ __forceinline__ void mma_i8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t"
      "}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* m, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(m), "r"(src), "r"(c0), "r"(c1)
               : "memory");
}
// All but the newest store that this thread committed have finished reading shared memory.
__device__ __forceinline__ void tma_store_wait_read_but_one() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }
}  // namespace ptx

// BN: the widest tile
template <int BN, typename OutT>
struct Int8PairCfg {
  static constexpr int kStageA = kBM * kBK, kStageB = BN / 2 * kBK;
  static constexpr int kEpiWarps = 8, kProducerWarp = 8, kMmaWarp = 9, kThreads = 320;
  static constexpr int kCols = BN / 2;                                // columns of an epilogue warp at most
  static constexpr int kBoxBytes = 32 * 32 * (int)sizeof(OutT);       // its 32 rows of 32 columns
  static constexpr int kStaging = kEpiWarps * 2 * kBoxBytes;          // two boxes a warp
  static constexpr int kScales = kEpiWarps * 2 * kCols * 4;           // sb and bias of its columns: no warp waits for another
  static constexpr int kFixed = kStaging + kScales + 1024 + 256;
  static constexpr int kFit = (232448 - kFixed) / (kStageA + kStageB), kStages = kFit < 8 ? kFit : 8;
  static constexpr int kTmemCols = BN == 256 ? 512 : 256, kAccStride = BN == 256 ? 256 : 128;
  static constexpr size_t kSmemBytes = (size_t)kStages * (kStageA + kStageB) + kFixed;
  static_assert(kStages * (kStageA + kStageB) >= 6 * 16384, "the sums of the other splits fit the ring");
};

template <int BN, bool SWAP, typename OutT>
__global__ void __launch_bounds__(Int8PairCfg<BN, OutT>::kThreads, 1)
int8_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                 const __grid_constant__ CUtensorMap tmap_c, const Int8Params p) {
  using Cfg = Int8PairCfg<BN, OutT>;
  constexpr int S = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_al = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
  const uint32_t sA = smem_base, sB = smem_base + S * Cfg::kStageA;
  constexpr uint32_t kRing = S * (Cfg::kStageA + Cfg::kStageB);
  const uint32_t staging = smem_base + kRing;
  float* cols = reinterpret_cast<float*>(smem_al + kRing + Cfg::kStaging);  // [warp][2][kCols]: sb, bias
  uint64_t* bars = reinterpret_cast<uint64_t*>(cols + Cfg::kScales / 4);
  const uint32_t bar0 = ptx::smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (S + s); };
  auto tfull_bar = [&](int b) { return bar0 + 8u * (2 * S + b); };
  auto tempty_bar = [&](int b) { return bar0 + 8u * (2 * S + 2 + b); };
  const uint32_t sum_bar = bar0 + 8u * (2 * S + 4);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(bars + 2 * S + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * S + 6);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t cluster_rank = ptx::cluster_ctarank(), rank = cluster_rank & 1, leader_rank = cluster_rank - rank;
  const bool leader = rank == 0;
  const int bn = p.nt, splits = p.k_splits, ks = (int)cluster_rank >> 1;  // columns of the tile
  auto owner_of = [&](int chunk) { return (chunk >> 1) & (splits - 1); };  // K splits: the chunks of both halves go round

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      ptx::mbar_init(full_bar(s), 2);
      ptx::mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(tfull_bar(b), 1);
      ptx::mbar_init(tempty_bar(b), 2 * Cfg::kEpiWarps);
    }
    ptx::mbar_init(sum_bar, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    if (splits > 1) {  // the other splits' sums of this CTA's chunks
      int mine = 0;
      for (int j = 0; j < bn / 32; ++j) mine += owner_of(j) == ks;
      ptx::mbar_expect_tx(sum_bar, (uint32_t)(mine * (splits - 1) * 32 * kBM * 4));
    }
  }
  if (warp == Cfg::kMmaWarp) {
    ptx::tmem_alloc_pair(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), Cfg::kTmemCols);
    ptx::tmem_relinquish_pair();
  }
  if (warp == Cfg::kProducerWarp && lane == 0) {
    ptx::prefetch_tensormap(&tmap_a);
    ptx::prefetch_tensormap(&tmap_b);
    ptx::prefetch_tensormap(&tmap_c);
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_arrive_relaxed();  // waited for below: the peer's barriers are initialised before anything signals them
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_launch_dependents();
  // a cluster takes one tile where K is split, else as many as there are
  const int pair = (blockIdx.x >> 1) / splits, npairs = (gridDim.x >> 1) / splits, tiles = p.m_tiles * p.n_tiles;
  const int kb0 = ks * p.kb_per_split, kb1 = min(p.num_kb, kb0 + p.kb_per_split);
  auto coords = [&](int t, int& mt, int& nt) { tile_coords(t, p.m_tiles, p.n_tiles, p.group_m, p.per_group_div, mt, nt); };
  // What is read and overwritten below belongs to the kernels before, which may still run; the weights of the first K blocks are
  // asked for all the same, as a prefetch into L2, a row each.
  if ((int)threadIdx.x < (SWAP ? kBM : bn / 2)) {
    int mt, nt;
    coords(pair, mt, nt);
    const int row = (SWAP ? mt * 2 * kBM + (int)rank * kBM : nt * bn + (int)rank * (bn / 2)) + (int)threadIdx.x;
    if (row < p.N)
      prefetch_weight_row(reinterpret_cast<const uint8_t*>(p.w) + (int64_t)row * p.w_ld + kb0 * kBK, min(kPrefetchKb, kb1 - kb0));
  }
  __syncwarp();
  ptx::cluster_wait();
  grid_dependency_wait();

  if (warp == Cfg::kProducerWarp) {
    if (ptx::elect_one()) {
      const uint32_t bytes = Cfg::kStageA + bn / 2 * kBK;
      int s = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += npairs) {
        int mt, nt;
        coords(t, mt, nt);
        const int a_row = mt * 2 * kBM + (int)rank * kBM, b_row = nt * bn + (int)rank * (bn / 2);
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = ptx::mbar_wait(empty_bar(s), phase, abort_flag);
          if (!ok) break;
          const uint32_t lf = ptx::mapa(full_bar(s), leader_rank);
          ptx::mbar_expect_tx_cluster(lf, bytes);
          ptx::tma_load_2d_pair(sA + s * Cfg::kStageA, &tmap_a, kb * kBK, a_row, lf);
          ptx::tma_load_2d_pair(sB + s * Cfg::kStageB, &tmap_b, kb * kBK, b_row, lf);
          if (++s == S) s = 0, phase ^= 1;
        }
      }
      // the leader's last arrivals on this CTA's empty barriers, before its shared memory may go
      for (int i = 0; i < S && ok; ++i) {
        ok = ptx::mbar_wait(empty_bar(s), phase, abort_flag);
        if (++s == S) s = 0, phase ^= 1;
      }
    }
    __syncwarp();
  } else if (warp == Cfg::kMmaWarp) {
    if (leader && ptx::elect_one()) {
      const uint32_t idesc = ptx::idesc_s8_s32(2 * kBM, bn);
      const uint16_t both = (uint16_t)(3u << leader_rank);
      const uint64_t da0 = ptx::smem_desc_sw128(sA), db0 = ptx::smem_desc_sw128(sB);
      int s = 0, b = 0;
      uint32_t phase = 0, tphase = 1;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += npairs) {
        ok = ptx::mbar_wait(tempty_bar(b), tphase, abort_flag);
        const uint32_t d = tmem_base + b * Cfg::kAccStride;
#pragma unroll 1
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
          ok = ptx::mbar_wait(full_bar(s), phase, abort_flag);
          if (!ok) break;
          ptx::tc_fence_after();
          // a stage further = its bytes >> 4 in the address field, which does not overflow: shared memory ends below 2^18
          const uint64_t da = da0 + (uint32_t)(s * (Cfg::kStageA >> 4)), db = db0 + (uint32_t)(s * (Cfg::kStageB >> 4));
#pragma unroll
          for (int k = 0; k < kBK / 32; ++k) ptx::mma_i8_pair(d, da + 2 * k, db + 2 * k, idesc, kb > kb0 || k > 0);
          ptx::mma_commit_pair_multicast(empty_bar(s), both);
          if (++s == S) s = 0, phase ^= 1;
        }
        if (!ok) break;
        ptx::mma_commit_pair_multicast(tfull_bar(b), both);
        if (++b == 2) b = 0, tphase ^= 1;
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t leader_tempty = ptx::mapa(tempty_bar(0), leader_rank);
    float* my_cols = cols + warp * 2 * Cfg::kCols;
    const uint32_t boxes = staging + warp * 2 * Cfg::kBoxBytes;
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const int chunks = bn / 32;
    int b = 0, box_no = 0;
    uint32_t phase = 0;
    for (int t = pair; t < tiles; t += npairs) {
      int mt, nt;
      coords(t, mt, nt);
      const int row0 = mt * 2 * kBM + (int)rank * kBM + quarter * 32, row = row0 + lane;
      // scale (and bias) of this thread's row and of the tile's columns
      auto load_bias = [&](int n) { return p.bias != nullptr ? to_f32<OutT>(static_cast<const OutT*>(p.bias)[n]) : 0.f; };
      float own = 0.f, own_bias = 0.f;
      if (row < (SWAP ? p.N : p.M)) {
        own = ld_operand((SWAP ? p.sb : p.sa) + row);
        if (SWAP) own_bias = load_bias(row);
      }
      __syncwarp();  // the last tile's columns have been read
      for (int j = half; j < chunks; j += 2) {
        const int n = nt * bn + j * 32 + lane, at = (j >> 1) * 32 + lane;
        const bool inside = n < (SWAP ? p.M : p.N);
        my_cols[at] = inside ? ld_operand((SWAP ? p.sa : p.sb) + n) : 0.f;
        if (!SWAP) my_cols[Cfg::kCols + at] = inside ? load_bias(n) : 0.f;
      }
      __syncwarp();
      bool ok = ptx::mbar_wait(tfull_bar(b), phase, abort_flag);
      if (!ok && splits == 1) break;
      ptx::tc_fence_after();
      const uint32_t ta = lane_base + b * Cfg::kAccStride;
      // K splits. Slot of a sum: [chunk of its owner][source][4 columns][row], 16 bytes
      auto slot = [&](int j, int src) {
        const int mine = (j >> 1) / splits * 2 + half;
        return (uint32_t)(((mine * (splits - 1) + src) * 8 * kBM + quarter * 32 + lane) * 16);
      };
      if (splits > 1) {
        __syncwarp();
        ptx::cluster_arrive_relaxed();
        ptx::cluster_wait();  // every ring is idle
        for (int j = half; j < chunks; j += 2) {
          const int owner = owner_of(j);
          if (owner == ks) continue;
          uint32_t v[32];
          ptx::tmem_ld32(ta + j * 32, v);
          ptx::tmem_ld_wait(v);
          const uint32_t cta = (uint32_t)owner * 2 + rank, dst = ptx::mapa(smem_base + slot(j, ks < owner ? ks : ks - 1), cta),
                         bar = ptx::mapa(sum_bar, cta);
#pragma unroll
          for (int g = 0; g < 8; ++g)
            ptx::st_async_v4(dst + g * kBM * 16, v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3], bar);
        }
        ok = ok && ptx::mbar_wait_cluster(sum_bar, 0, abort_flag);
      }
#pragma unroll 1
      for (int j = half; j < chunks; j += 2) {
        if (splits > 1 && (owner_of(j) != ks || !ok)) continue;
        uint32_t v[32];
        ptx::tmem_ld32(ta + j * 32, v);
        ptx::tmem_ld_wait(v);
        for (int src = 0; src < splits - 1; ++src) {
          const uint32_t from = smem_base + slot(j, src);
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const int4 o = ptx::ld_shared_i4(from + g * kBM * 16);
            v[4 * g] += o.x, v[4 * g + 1] += o.y, v[4 * g + 2] += o.z, v[4 * g + 3] += o.w;
          }
        }
        const uint32_t box = boxes + (box_no & 1) * Cfg::kBoxBytes;
        ++box_no;
        if (lane == 0) ptx::tma_store_wait_read_but_one();  // the box before the last has left this half of the staging area
        __syncwarp();
        const float* col = my_cols + (j >> 1) * 32;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float f[8];
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            const uint32_t* q = v + 8 * g + i;
            const float4 c4 = ld_shared_f4(col + 8 * g + i);
            if constexpr (SWAP) {
              f[i + 0] = fmaf((float)(int)q[0] * c4.x, own, own_bias);
              f[i + 1] = fmaf((float)(int)q[1] * c4.y, own, own_bias);
              f[i + 2] = fmaf((float)(int)q[2] * c4.z, own, own_bias);
              f[i + 3] = fmaf((float)(int)q[3] * c4.w, own, own_bias);
            } else {
              const float4 b4 = ld_shared_f4(col + Cfg::kCols + 8 * g + i);
              f[i + 0] = fmaf((float)(int)q[0] * own, c4.x, b4.x);
              f[i + 1] = fmaf((float)(int)q[1] * own, c4.y, b4.y);
              f[i + 2] = fmaf((float)(int)q[2] * own, c4.z, b4.z);
              f[i + 3] = fmaf((float)(int)q[3] * own, c4.w, b4.w);
            }
          }
          // the box has rows of 64 bytes (16-bit types) or 128, tokens, in the swizzle of the tensor map
          constexpr int kRow = 32 * (int)sizeof(OutT), kXor = kRow / 16 - 1, kShift = kRow == 64 ? 1 : 0;
          if constexpr (SWAP) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int t = 8 * g + i, byte = lane * (int)sizeof(OutT);
              const OutT o = from_f32<OutT>(f[i]);
              const uint32_t at = box + t * kRow + (((byte >> 4) ^ ((t >> kShift) & kXor)) << 4) + (byte & 15);
              if constexpr (sizeof(OutT) == 2)
                asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"(*reinterpret_cast<const uint16_t*>(&o)) : "memory");
              else
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(o) : "memory");
            }
          } else if constexpr (sizeof(OutT) == 2) {
            const uint4 o = pack8<OutT>(f);
            const uint32_t at = box + lane * kRow + ((g ^ ((lane >> kShift) & kXor)) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(o.x), "r"(o.y), "r"(o.z), "r"(o.w) : "memory");
          } else {
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
              const uint32_t at = box + lane * kRow + (((2 * g + i / 4) ^ (lane & kXor)) << 4);
              asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(f[i]), "f"(f[i + 1]), "f"(f[i + 2]), "f"(f[i + 3]) : "memory");
            }
          }
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          const int col0 = nt * bn + j * 32;
          const int channel = SWAP ? row0 : col0, token = SWAP ? col0 : row0;
          if (token < p.M && channel < p.N) ptx::tma_store_2d(&tmap_c, box, channel, token);
          ptx::tma_store_commit();
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      // The accumulator is in registers. Only for a tile that waits for it: nobody would wait for the last ones, and the follower's could
      // then reach the leader's shared memory after the leader has left it.
      if (lane == 0 && t + 2 * npairs < tiles) ptx::mbar_arrive_cluster(leader_tempty + 8 * b);
      if (++b == 2) b = 0, phase ^= 1;
    }
    if (lane == 0) ptx::tma_store_wait_all();
  }
  if (splits > 1 && warp >= Cfg::kEpiWarps) {  // the other warps' share of the cluster barrier above
    __syncwarp();
    ptx::cluster_arrive_relaxed();
    ptx::cluster_wait();
  }

  if (*abort_flag) {
    const unsigned long long t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_arrive_relaxed();
  // Neither CTA leaves while the other may still signal its barriers or read its shared memory: every such signal has been waited for by
  // then (this barrier itself orders nothing), and it holds a CTA back until its peer's waits are done, too.
  ptx::cluster_wait();
  if (threadIdx.x == 0 && *abort_flag) atomicCAS(p.status, 0, 1);
  if (warp == Cfg::kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem_base, Cfg::kTmemCols);
  }
}

// p.nt columns per tile (a multiple of 32, at most BN), p.k_splits 1, 2 or 4.
template <int BN, bool SWAP, typename OutT>
inline int launch_int8_pair(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t K, Int8Params p, cudaStream_t st) {
  using Cfg = Int8PairCfg<BN, OutT>;
  const int64_t rows = SWAP ? p.N : p.M, cols = SWAP ? p.M : p.N;
  p.m_tiles = (int)cdiv(rows, 2 * kBM);
  p.n_tiles = (int)cdiv(cols, p.nt);
  p.kb_per_split = (int)cdiv(p.num_kb, p.k_splits);
  p.group_m = row_group(rows, K, 2 * kBM);
  p.per_group_div = make_fastdiv(p.group_m * p.n_tiles);
  CUtensorMap ta, tb, tc;
  if (int rc = encode_tmap_s8(&ta, SWAP ? B : A, rows, K, SWAP ? ldb : lda, kBM, "rows")) return rc;
  if (int rc = encode_tmap_s8(&tb, SWAP ? A : B, cols, K, SWAP ? lda : ldb, p.nt / 2, "columns")) return rc;
  const CUtensorMapDataType type = sizeof(OutT) == 4                                ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : std::is_same<OutT, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                              : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (int rc = encode_tmap(&tc, type, (int)sizeof(OutT), p.C, p.M, p.N, p.N, 32, 32, CU_TENSOR_MAP_L2_PROMOTION_NONE, "C")) return rc;
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
  const int slots = sm_count() / 2, pairs = (int)(p.k_splits > 1 || tiles < slots ? tiles : slots);
  auto k = int8_pair_kernel<BN, SWAP, OutT>;
  if (int rc = allow_smem(k, Cfg::kSmemBytes, "int8_pair_kernel")) return rc;
  return launch_dependent(k, dim3((unsigned)(2 * pairs * p.k_splits)), Cfg::kThreads, Cfg::kSmemBytes, st, 2u * p.k_splits,
                          "int8_pair_kernel", ta, tb, tc, p);
}

}  // namespace b200
