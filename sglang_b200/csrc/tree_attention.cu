// Attention of the newest tokens of every sequence (one, or a tree of drafted ones) over a paged cache:
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale * k_scale * log2(e),  m near the largest exponent so far
// The G query heads of a kv head times the new tokens are the rows of one problem, NT of them a tile. 128 keys fill the lanes of the tensor core's
// tile and the rows are its columns, so that few rows cost little:
//   S^T [128 keys, NT] = K Q^T     K and Q in shared memory, S^T in TMEM, two buffers
//   O^T [D, NT]       += V^T P^T   V as it lies in the cache (its rows are the product's depth), P^T [keys, NT] in shared memory
// A thread of the softmax has one key and the rows' columns. It takes its exponentials against a reference per row that is moved only when a score
// lies 2^8 above the one it was taken from, so a tile needs one vote of the threads and no maxima over keys; sums over keys stay in registers until the
// end. With more than 64 rows the rows fill the lanes and the keys are the columns, S [128, keys] and O [128, D], P in TMEM over its own S: a softmax row
// is a thread's own, and P needs no shared memory.
// Keys come by their pages' addresses, any page size, in 16-byte pieces by asynchronous copies; codes of an FP8 cache land in a ring of their own and
// become fp16 values, exactly, on their way into the ring of tiles. All tiles of all (sequence, kv head, row tile) form one line that is cut into equal
// pieces, one per CTA, so that ragged lengths leave no SM idle; rows whose keys were cut leave partial sums in a workspace, which a second kernel joins in
// the line's order.
// Few rows over a 16-bit cache are bound by its bytes: 128 sequences of up to 8192 tokens, 8 kv heads of 128, one token a page, 2.17 GB: 333 us, 6.5 TB/s; 16 of up
// to 16384 with 8 drafted tokens, 64 query heads (64 rows), 597 MB: 127 to 131 us, 4.6 TB/s. An FP8 cache is bound by the way of its codes through the SM, copied,
// read, widened and stored: 64 sequences of up to 16384, one token, 1.08 GB: 238 to 242 us, 4.5 TB/s. 128 rows by the exponentials, 16 a clock and SM, and by the
// latency of the steps between two products: 61 sequences of up to 32768, 16 tokens, FP8, 264 MB: 113 to 119 us, 540 TFLOP/s.
#include <cfloat>

#include "gemm_host.cuh"
#include "int8_round.cuh"

namespace b200 {
namespace ptx {

// Descriptor of an operand in shared memory whose upper half is known at compile time: it takes one register, and steps are 32-bit additions.
struct Operand {
  uint32_t low, high;
  __device__ __forceinline__ Operand at(uint32_t bytes) const { return {low + (bytes >> 4), high}; }
};
// Rows of 128 bytes along the depth (K-major), 128-byte swizzle, groups of eight rows one behind the other
__device__ __forceinline__ Operand operand_sw128(uint32_t addr) {
  return {(addr >> 4) | (1u << 16), (uint32_t)(1024 >> 4) | (1u << 14) | (2u << 29)};
}
// Rows that are the depth: ROW bytes (32, 64 or 128: that swizzle) across, groups of eight rows one behind the other, the next ROW / 2 elements across `block`
// bytes further
template <int ROW>
__device__ __forceinline__ Operand operand_depth_rows(uint32_t addr, uint32_t block) {
  return {(addr >> 4) | ((block >> 4) << 16), (uint32_t)(8 * ROW >> 4) | (1u << 14) | ((ROW == 128 ? 2u : ROW == 64 ? 4u : 6u) << 29)};
}
// D (+)= A B with 16-bit operands in shared memory, fp32 sums
__device__ __forceinline__ void mma_f16(uint32_t d, Operand a, Operand b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 a, {%1, %2};\n\t"
      "mov.b64 b, {%3, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t"
      "}" ::"r"(d),
      "r"(a.low), "r"(a.high), "r"(b.low), "r"(b.high), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The same with A in TMEM, two elements a column
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, Operand b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b64 b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t"
      "}" ::"r"(d),
      "r"(a), "r"(b.low), "r"(b.high), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor for kind::f16, fp32 sums: bits 4-5 D format (1 = f32), 7-9 / 10-12 A / B format (0 = f16, 1 = bf16), 15 / 16 rows of A / B are
// the depth (depth_rows: 1, 2), 17-22 N >> 3, 24-28 M >> 4
__host__ __device__ constexpr uint32_t idesc_f16_f32(bool bf16, uint32_t depth_rows, int M, int N) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | (depth_rows << 15) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
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
// Arrives once all copies that this thread has issued so far have landed
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void st_shared_16(uint32_t dst, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint32_t ld_byte(const uint8_t* p) {
  uint32_t v;
  asm volatile("ld.global.u8 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Moves this warp's registers from what it was launched with to N a thread (all warps of its group of four do the same)
template <int N, int LAUNCH>
__device__ __forceinline__ void give_registers() {
  if constexpr (N > LAUNCH) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
  if constexpr (N < LAUNCH) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
// Two fp32 operations at once
__device__ __forceinline__ void fma_two(float& a, float& b, float x0, float x1, float y0, float y1, float z0, float z1) {  // x y + z
  asm("{.reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%6, %7}; fma.rn.f32x2 x, x, y, z; mov.b64 {%0, %1}, x;}"
      : "=f"(a), "=f"(b)
      : "f"(x0), "f"(x1), "f"(y0), "f"(y1), "f"(z0), "f"(z1));
}
__device__ __forceinline__ void add_two(float& a, float& b, float x0, float x1) {  // a += x0, b += x1
  asm("{.reg .b64 x, y; mov.b64 x, {%0, %1}; mov.b64 y, {%2, %3}; add.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x;}" : "+f"(a), "+f"(b) : "f"(x0), "f"(x1));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// true in all `threads` threads of barrier `id` if it is in one
__device__ __forceinline__ bool any_of(int id, int threads, bool mine) {
  uint32_t all;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.b32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t"
      "}"
      : "=r"(all)
      : "r"(id), "r"(threads), "r"((uint32_t)mine)
      : "memory");
  return all != 0;
}
__device__ __forceinline__ uint4 ld_shared_16(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
  return v;
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

constexpr int kKeys = 128;  // of a tile
__device__ const uint4 not_a_number16 = {0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};  // in either 16-bit type
__device__ const uint4 not_a_number8 = {0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu};

template <int D, int NT, bool FP8>
struct AttnCfg {
  static constexpr int kWidth = D < 128 ? D : 128, kParts = D / kWidth;  // elements of a head in a stage; stages of a tile of keys, or of values
  static constexpr int kStage = kKeys * kWidth * 2;
  // What the two groups of softmax warps share: up to 32 rows they take the tiles in turn, each with an O of its own, so that one computes while the other
  // waits for its products; with 64 each has half of the rows of every tile; with 128 the rows are in the lanes, P lies in TMEM over its own S, and each has
  // half of the keys of every tile, for all rows, and an O of its own.
  static constexpr bool kRowsInLanes = NT == 128, kTurns = NT <= 32, kTwoO = NT != 64;
  static constexpr int kCols = kTurns ? NT : NT / 2;  // columns of a softmax thread
  static constexpr int kQBytes = NT * D * 2, kPBytes = kRowsInLanes ? 0 : kKeys * NT * 2;
  // fp32 words per row: scales of the rows of four row tiles, references, factors, sums per warp, tokens, rows of the output; or bits per 32 keys, for both
  // groups, of two tiles
  static constexpr int kTables = NT * 4 * (kRowsInLanes ? 4 + 2 + 2 + 16 : 4 + 2 + 2 + 8 + 2 + 1);
  // Warps: two groups of four for the softmax; one issues the output's products, two bring queries, one issues the scores' products; then four that bring keys
  // and four values, or all bring both: eight where an FP8 cache's ring is short, so that a stage is soon widened, four with two stages a tile
  static constexpr int kSoftmaxWarps = 8, kOutputWarp = kSoftmaxWarps, kQWarp = kOutputWarp + 1, kScoreWarp = kOutputWarp + 3, kProducerWarp = kOutputWarp + 4;
  // (Up to 32 rows the queries of the next row tile are brought while this one ends; more rows take so many loads that the softmax warps, which have
  // nothing to do until then, bring them themselves: 128 rows 14 thousand clocks by three warps)
  static constexpr bool kQueryWarps = NT <= 32;
  static constexpr bool kSplit = kParts == 1 && (!FP8 || NT <= 32);
  static constexpr int kProducerWarps = kParts == 1 ? 8 : 4, kWarpKeys = kParts == 1 && !kSplit ? 16 : 32;  // keys of a stage that a warp brings
  static constexpr int kThreads = (kProducerWarp + kProducerWarps) * 32;
  // FP8: codes land in a ring of each producer's own, kRaw stages deep, and go from there into the ring of 16-bit tiles
  static constexpr int kRawStage = kWarpKeys * kWidth, kRaw = !FP8 ? 0 : kSplit ? 2 : 3, kRawBytes = kProducerWarps * kRaw * kRawStage;
  static constexpr int kFixed = kQBytes + 2 * kPBytes + kRawBytes + kTables + 1024 + 512;
  static constexpr int kFit = (232448 - kFixed) / kStage;
  // places for keys and for values: each have a ring of their own, so that a wait for a place is never for a phase two ahead
  static constexpr int kStages = kFit < 12 ? kFit : 12, kPlacesK = kStages / 2, kPlacesV = kStages - kPlacesK;
  // Registers of a thread at launch, and of the three kinds of warps
  static constexpr int kLaunchRegs = 65536 / kThreads / 8 * 8;
  static constexpr int kSoftmaxRegs = kParts == 1 ? 112 : 160, kProducerRegs = kParts == 1 ? 88 : 112, kOtherRegs = 80;
  static_assert((8 * kSoftmaxRegs + 4 * kOtherRegs + kProducerWarps * kProducerRegs) * 32 <= kThreads * kLaunchRegs,
                "the registers add up to no more than at launch");
  // TMEM columns: the scores of two tiles, then an O for each of the two groups
  static constexpr int kSCols = kRowsInLanes ? kKeys : NT, kOCols = kRowsInLanes ? D : kParts * NT, kTmemO = 2 * kSCols;
  static constexpr int kTmemUsed = 2 * kSCols + (kTwoO ? 2 : 1) * kOCols;
  static constexpr int kTmemCols = kTmemUsed <= 64 ? 64 : kTmemUsed <= 128 ? 128 : kTmemUsed <= 256 ? 256 : 512;
  static constexpr size_t kSmemBytes = (size_t)kFixed + (size_t)kStages * kStage;
  static_assert(kPlacesK >= 1 && kTmemUsed <= 512 && kSmemBytes <= 232448, "the rings fit");
};

// Sequence b as the kernel takes it: whatever the index tensors hold, tokens and keys stay inside q and the page table.
struct Seq {
  int start, n, len, row_tiles, key_tiles;
  // A row tile's length on the line: its tiles of keys, and as many more as its queries, masks and output cost (16 x 16384 keys, 8 tokens: without them the
  // CTAs with the short sequences took 156 us where others took 94)
  __device__ __forceinline__ int units(int extra) const { return key_tiles + extra; }
  __device__ __forceinline__ int64_t length(int heads, int extra) const { return n > 0 ? (int64_t)heads * row_tiles * units(extra) : 0; }
};
template <int NT>
constexpr int kExtraTiles = NT <= 32 ? 1 : 7;
template <int NT>
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
  s.row_tiles = (s.n * p.group + NT - 1) / NT;
  s.key_tiles = max(1, (s.len + kKeys - 1) / kKeys);
  return s;
}

// Where an offset on a sequence's part of the line lies: kv head, row tile, place in that row tile's length. In 64 bits: the row tiles of one head may be
// longer than 2^31 together.
struct LinePlace {
  int h, qt, at;
};
__host__ __device__ inline LinePlace line_place(int64_t offset, int row_tiles, int units) {
  const int64_t tile = offset / units, head = tile / row_tiles;
  return {(int)head, (int)(tile - head * row_tiles), (int)(offset - tile * units)};
}

// A CTA's piece of the line, one (sequence, head, row tile) at a time
template <int NT>
struct Walk {
  const AttnParams& p;
  int b, h, qt, t0, t1;  // sequence, kv head, row tile; its tiles of keys t0 .. t1 - 1
  int at, end;           // the piece's part of the row tile's length
  int64_t left;          // of the piece
  Seq s;
  __device__ __forceinline__ Walk(const AttnParams& p_, int b0, int64_t offset, int64_t length) : p(p_), b(b0), left(length) {
    h = qt = t0 = t1 = at = end = 0;
    s = {};
    if (left <= 0) return;
    s = seq_of<NT>(p, b);
    const LinePlace place = line_place(offset, s.row_tiles, s.units(kExtraTiles<NT>));
    h = place.h, qt = place.qt, at = place.at;
    settle();
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ void next() {
    leave();
    settle();
  }

 private:
  __device__ __forceinline__ void settle() {  // to the next row tile of which the piece has keys
    while (left > 0) {
      end = (int)min((int64_t)s.units(kExtraTiles<NT>), at + left);
      t0 = max(0, at - kExtraTiles<NT>);
      t1 = max(0, end - kExtraTiles<NT>);
      if (t1 > t0) return;
      leave();
    }
  }
  __device__ __forceinline__ void leave() {
    left -= end - at;
    at = 0;
    if (left <= 0 || ++qt < s.row_tiles) return;
    qt = 0;
    if (++h < p.a.kv_heads) return;
    h = 0;
    do {
      s = seq_of<NT>(p, ++b);
    } while (s.n == 0 && b + 1 < p.a.sequences);
  }
};

// Four E4M3 codes as fp16 values: exact
__device__ __forceinline__ void widen4(uint32_t codes, uint32_t& low, uint32_t& high) {
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h;}" : "=r"(low), "=r"(high) : "r"(codes));
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

// A row's reference is taken this far below its largest score (in powers of two), and stays until a score exceeds it by kReach: most rows move theirs in the
// first tile alone. Weights in fp16 reach from 2^15 down to steps of 2^-24, so the largest stands at 2^7 or higher, and what a long context's many small
// weights lose is below 2^-32 of it each (with the reference at the largest score itself 2^-25: 131072 keys of 2^-26 each were lost, 2^-9 of the
// sum, which is taken of the fp32 weights). bf16 has the range of the sums.
template <typename M>
constexpr float kBelow = std::is_same_v<M, __half> ? 7.f : 0.f;
template <typename M>
constexpr float kReach = kBelow<M> + 8.f;
constexpr float kNothing = -INFINITY;  // in the place of a group's factor for a row of which it has seen nothing
constexpr float kNoRef = 3e38f;  // of a row that has seen nothing yet, negated like all references: any score exceeds it, and -infinity stays what it is

// Value i of lane l, N <= 32 of them in each of 32 lanes -> lane l has the result over all lanes of value l % N. Each step halves the values that a
// lane still has, N - 1 exchanges and 5 - log2 N more.
template <int N, int BIT = 1, typename F>
__device__ __forceinline__ float across_lanes(const float (&v)[N], F op) {
  if constexpr (BIT == 32) {
    return v[0];
  } else if constexpr (N == 1) {
    const float next[1] = {op(v[0], __shfl_xor_sync(0xffffffffu, v[0], BIT))};
    return across_lanes<1, BIT * 2>(next, op);
  } else {
    const bool upper = (threadIdx.x & BIT) != 0;
    float next[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float other = __shfl_xor_sync(0xffffffffu, upper ? v[2 * i] : v[2 * i + 1], BIT);
      next[i] = op(upper ? v[2 * i + 1] : v[2 * i], other);
    }
    return across_lanes<N / 2, BIT * 2>(next, op);
  }
}

constexpr int kBothGroups = 3;  // barrier of both groups of softmax warps

// A piece of a row tile as its odd values need it: its sequence's own keys [j0, j1)
struct OddPiece {
  int b, h, qt, start, rows, prefix, j0, j1;
  bool whole;
  int64_t slot0;
};
// Values that are not finite and were taken out go to the rows that see them, whatever their weight. 32 keys at a time the warps find out which rows see each,
// then a thread with an element of the head notes which rows take what of it, and each row's element is changed once at the end. (A change for every key
// would cost keys times rows trips to memory, more than the other warps wait for where a long prompt's values are NaN. Apart from the kernel, whose registers
// it would take.)
template <typename T, int D, int NT, bool FP8>
__device__ __noinline__ void add_odd_values(const AttnParams& p, const OddPiece& s, uint32_t* rows_of_key /* [32][kWords] */) {
  const b200_tree_attention_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr uint32_t kExponent = std::is_same_v<T, __nv_bfloat16> && !FP8 ? 0x7f80u : 0x7c00u;
  constexpr int kWords = NT <= 32 ? 1 : NT / 32, kPer = 4 * kWords;  // words of a key; keys that a warp looks at
  uint32_t nan[kWords] = {}, plus[kWords] = {}, minus[kWords] = {};   // rows that take one
  const int d = threadIdx.x, my_row = warp % kWords * 32 + lane, my_token = fast_div(s.qt * NT + min(my_row, s.rows - 1), p.group_div);
  const uint8_t* const line_of_mask = static_cast<const uint8_t*>(a.mask) + (int64_t)(s.start + my_token) * a.mask_ld;
#pragma unroll 1
  for (int j0 = s.j0; j0 < s.j1; j0 += 32) {
#pragma unroll 4
    for (int i = 0; i < kPer; ++i) {
      const int k = warp / kWords * kPer + i, own = j0 + k - s.prefix;
      const bool sees = my_row < s.rows && j0 + k < s.j1 && (a.mask ? own < a.mask_width && ptx::ld_byte(line_of_mask + own) != 0 : own <= my_token);
      const uint32_t all = __ballot_sync(0xffffffffu, sees);
      if (lane == 0) rows_of_key[k * kWords + warp % kWords] = all;
    }
    int64_t my_value = -1;  // of key j0 + lane: where it begins, if the cache has its page
    if (j0 + lane < s.j1) {
      const int page = fast_div(j0 + lane, p.page_div), entry = ld_operand(a.page_table + (int64_t)s.b * a.page_table_ld + page);
      if (entry >= 0 && entry < a.pages) my_value = entry * a.v_page + (j0 + lane - page * a.page_size) * a.v_token + s.h * a.v_head;
    }
    ptx::any_of(kBothGroups, 256, false);
#pragma unroll 8
    for (int k = 0; k < 32; ++k) {
      const int64_t value = __shfl_sync(0xffffffffu, my_value, k);
      uint32_t x = 0;
      if (value >= 0 && d < D) {
        if constexpr (FP8) x = (static_cast<const volatile uint8_t*>(a.v_cache)[value + d] & 0x7fu) == 0x7fu ? kExponent + 1 : 0u;
        else x = static_cast<const volatile uint16_t*>(a.v_cache)[value + d];
      }
      if ((x & kExponent) != kExponent) continue;  // finite
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const uint32_t to = rows_of_key[k * kWords + i];
        if ((x & 0x7fffu) > kExponent) nan[i] |= to;
        else if (x & 0x8000u) minus[i] |= to;
        else plus[i] |= to;
      }
    }
    ptx::any_of(kBothGroups, 256, false);
  }
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    const uint32_t take = nan[i] | plus[i] | minus[i], none = nan[i] | (plus[i] & minus[i]);
    for (uint32_t left = take; left != 0; left &= left - 1) {
      const int bit = __ffs(left) - 1, n = i * 32 + bit;
      const float v = (none >> bit) & 1u ? NAN : (minus[i] >> bit) & 1u ? -INFINITY : INFINITY;
      const int at = s.qt * NT + n, token = fast_div(at, p.group_div);
      if (s.whole) {
        T* const o = static_cast<T*>(a.out) + ((int64_t)(s.start + token) * a.q_heads + s.h * p.group + at - token * p.group) * D + d;
        *o = from_f32<T>(to_f32<T>(*o) + v);
      } else {
        p.part_o[AttnCfg<D, NT, FP8>::kRowsInLanes ? s.slot0 * D + ((d >> 2) * p.row_slots + n) * 4 + (d & 3) : (s.slot0 + n) * D + d] += v;
      }
    }
  }
}

template <typename T, int D, int NT, bool FP8>
__global__ void __launch_bounds__(AttnCfg<D, NT, FP8>::kThreads, 1) tree_attention_kernel(const __grid_constant__ AttnParams p) {
  using Cfg = AttnCfg<D, NT, FP8>;
  // Weights are rounded to the 16 bits that the tensor core multiplies with the values; their sum is taken of the fp32 ones. (An output so differs from that
  // of fp32 weights by less than its own rounding: 2.2e-3 against 1.7e-3 off in bf16, root mean square.)
  // An FP8 cache is multiplied in fp16, which holds its codes, whatever the queries' type: a code is converted by one instruction for two, and weights keep
  // 11 bits. bf16 queries become fp16 behind a power of two per row that brings their largest element to 2^7 .. 2^8; what then lies below fp16's
  // normal range is 2^-21 of it.
  using M = std::conditional_t<FP8, __half, T>;
  constexpr bool kRowScales = FP8 && std::is_same_v<T, __nv_bfloat16>, kBf16 = std::is_same_v<M, __nv_bfloat16>;
  constexpr uint32_t kExponent = kBf16 ? 0x7f80u : 0x7c00u;
  constexpr int S = Cfg::kStages, kParts = Cfg::kParts;
  const b200_tree_attention_args& a = p.a;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_al = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
  constexpr uint32_t kRing = S * Cfg::kStage;
  const uint32_t sKV = smem_base, sQ = smem_base + kRing, sP = sQ + Cfg::kQBytes, sRaw = sP + 2 * Cfg::kPBytes;
  float* row_scale = reinterpret_cast<float*>(smem_al + kRing + Cfg::kQBytes + 2 * Cfg::kPBytes + Cfg::kRawBytes);  
  // [4][NT]: of a row tile's rows. Queries are brought as soon as the last scores of the row tile before have been asked for, which may be while the softmax
  // is still at the last tile of the one before that: three row tiles' scales are alive at a time
  float* minus_ref = row_scale + 4 * NT;                                                           // [2][NT]: of each group
  float* factor = minus_ref + 2 * NT;                                                              // [2][NT]
  float* by_warp = factor + 2 * NT;                                                                // [8][NT]
  int* token_of = reinterpret_cast<int*>(by_warp + 8 * NT);                                        // [2][NT]
  int* out_row = token_of + 2 * NT;                                                                // [NT]
  uint32_t* seen_words = reinterpret_cast<uint32_t*>(factor);                                      // rows in lanes: [2][2][NT][4], behind [2][NT] sums
  if (Cfg::kRowsInLanes) by_warp = factor, seen_words = reinterpret_cast<uint32_t*>(factor + 2 * NT);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_al + kRing + Cfg::kQBytes + 2 * Cfg::kPBytes + Cfg::kRawBytes + Cfg::kTables);
  const uint32_t bar0 = ptx::smem_u32(bars);
  auto full_bar = [&](uint32_t s) { return bar0 + 8u * s; };
  auto empty_bar = [&](uint32_t s) { return bar0 + 8u * (S + s); };
  struct Place {
    uint32_t at, phase;
  };
  auto place_of = [](int values, uint32_t n) {  // of the n-th stage of keys, or of values
    constexpr uint32_t kK = Cfg::kPlacesK, kV = Cfg::kPlacesV;
    return values ? Place{kK + n % kV, n / kV} : Place{n % kK, n / kK};
  };
  const uint32_t q_full = bar0 + 8u * (2 * S), q_empty = q_full + 8u;
  auto o_done = [&](uint32_t i) { return q_full + 16u + 8u * (i & 1); };  // products with the values of tiles i, i + 2, ..
  auto s_full = [&](uint32_t i) { return q_full + 32u + 8u * (i & 1); };
  auto p_full = [&](uint32_t i) { return q_full + 48u + 8u * (i & 1); };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(bars + 2 * S + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * S + 9);
  volatile int* begin_seq = abort_flag + 1;
  volatile int64_t* line = reinterpret_cast<volatile int64_t*>(bars + 2 * S + 10);  // offset within the first sequence, length of this CTA's piece, of every piece
  volatile int64_t* sums = line + 3;                                                // of each warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      ptx::mbar_init(full_bar(s), FP8 ? 128 / Cfg::kWarpKeys : 128);  // warps that have stored, or threads whose copies have landed
      ptx::mbar_init(empty_bar(s), 1);
    }
    ptx::mbar_init(q_full, Cfg::kQueryWarps ? 2 : Cfg::kSoftmaxWarps);
    ptx::mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(o_done(i), 1);
      ptx::mbar_init(s_full(i), 1);
      ptx::mbar_init(p_full(i), Cfg::kTurns ? 4 : 8);
    }
    *abort_flag = 0;
    *begin_seq = 0;
    line[0] = line[1] = 0;
    line[2] = 1;
    ptx::fence_mbar_init();
  }
  if (warp == Cfg::kOutputWarp) {
    ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), Cfg::kTmemCols);
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
    for (int b = b0; b < b1; ++b) mine += seq_of<NT>(p, b).length(a.kv_heads, kExtraTiles<NT>);
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
        const int64_t n = seq_of<NT>(p, b).length(a.kv_heads, kExtraTiles<NT>);
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
  Walk<NT> w(p, *begin_seq, line[0], line[1]);
  bool ok = true;

  // Query rows of the present row tile, those behind the last one as zeros; this warp's share of `lanes` threads begins at `first`
  auto load_queries = [&](int first, int lanes, int seg) {
    constexpr int kPerRow = D / 8, kAtOnce = Cfg::kQueryWarps ? 4 : 8;
    const int rows = min(NT, w.s.n * p.group - w.qt * NT);
#pragma unroll 1
    for (int from = first; from < NT * kPerRow; from += kAtOnce * lanes) {
      uint4 v[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int i = from + lane + u * lanes, r = min(i / kPerRow, rows - 1), c = i % kPerRow, at = w.qt * NT + r, token = fast_div(at, p.group_div);
        v[u] = ld_stream_16(static_cast<const T*>(a.q) + (int64_t)(w.s.start + token) * a.q_token + (w.h * p.group + at - token * p.group) * a.q_head + c * 8);
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int i = from + lane + u * lanes, r = i / kPerRow, c = i % kPerRow;
        if (r >= rows) v[u] = make_uint4(0, 0, 0, 0);
        if constexpr (kRowScales) {
          const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&v[u]);
          float top = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) top = fmaxf(top, fmaxf(fabsf(__low2float(x[k])), fabsf(__high2float(x[k]))));
#pragma unroll
          for (int o = kPerRow / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          // (134 - 254 at least; rows far below 1 have no score that is not 0, and the power's own inverse stays a normal number)
          const int e = top > 0.f && top < INFINITY ? min(134 - (int)(__float_as_uint(top) >> 23), 100) : 0;
          const float by = __uint_as_float((uint32_t)(127 + e) << 23);
          if (c == 0 && r < NT) row_scale[(seg & 3) * NT + r] = __uint_as_float((uint32_t)(127 - e) << 23);
          v[u] = make_uint4(pack2<__half>(__low2float(x[0]) * by, __high2float(x[0]) * by), pack2<__half>(__low2float(x[1]) * by, __high2float(x[1]) * by),
                            pack2<__half>(__low2float(x[2]) * by, __high2float(x[2]) * by), pack2<__half>(__low2float(x[3]) * by, __high2float(x[3]) * by));
        }
        if (r < NT) ptx::st_shared_16(sQ + (c >> 3) * (NT * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4), v[u]);
      }
    }
  };

  if (warp >= Cfg::kProducerWarp) {
    // ------------------------------------------------------------------ keys and values into the ring, a tile's keys, then its values
    ptx::give_registers<Cfg::kProducerRegs, Cfg::kLaunchRegs>();
    constexpr int kWarpKeys = Cfg::kWarpKeys;
    const int row0 = (warp - Cfg::kProducerWarp) * kWarpKeys % kKeys;  // this warp's keys of a tile, lane l has the addresses of the l-th
    // stages of a tile that are this warp's
    constexpr int kMine = Cfg::kSplit ? kParts : 2 * kParts;
    const int first_part = Cfg::kSplit && warp >= Cfg::kProducerWarp + 4 ? kParts : 0;
    constexpr int kPieces = Cfg::kWidth / (FP8 ? 16 : 8);  // of 16 bytes, of a key's part in the cache
    constexpr int kKeysAtOnce = 32 / kPieces;              // of a load of the warp
    constexpr int kSteps = kPieces * kWarpKeys / 32;
    constexpr int es = FP8 ? 1 : 2;
    auto entry_of = [&](const Walk<NT>& at, int t) {
      const int j = t * kKeys + row0 + lane;
      if (!at.more() || j >= at.s.len || lane >= kWarpKeys) return -1;
      return (int)ld_operand(a.page_table + (int64_t)at.b * a.page_table_ld + fast_div(j, p.page_div));
    };
    // this lane's key and its value; something readable where there is none. Warps that bring one of them know that one alone.
    const uint8_t* from[Cfg::kSplit ? 1 : 2];
    const bool values = Cfg::kSplit && first_part > 0;
    uint32_t absent, unknown;     // a bit per lane: no key there; a page that the cache does not have
    int t = w.t0, entry = entry_of(w, t);
    auto next_tile = [&] {
      const int j = t * kKeys + row0 + lane, in_page = j - fast_div(j, p.page_div) * a.page_size;
      const bool key = j < w.s.len && lane < kWarpKeys, page = entry >= 0 && entry < a.pages;
      absent = __ballot_sync(0xffffffffu, !key && lane < kWarpKeys);
      unknown = __ballot_sync(0xffffffffu, key && !page);
      const uint8_t* const some = static_cast<const uint8_t*>(a.q);
      const bool have = key && page;
      from[0] = have ? static_cast<const uint8_t*>(values ? a.v_cache : a.k_cache) +
                           (entry * (values ? a.v_page : a.k_page) + in_page * (values ? a.v_token : a.k_token) + w.h * (values ? a.v_head : a.k_head)) * es
                     : some;
      if constexpr (!Cfg::kSplit)
        from[1] = have ? static_cast<const uint8_t*>(a.v_cache) + (entry * a.v_page + in_page * a.v_token + w.h * a.v_head) * es : some;
      if (++t == w.t1) {
        w.next();
        t = w.t0;
      }
      entry = entry_of(w, t);
    };
    auto place = [&](uint32_t n) {  // of this warp's n-th stage
      const int part = first_part + n % kMine;
      return place_of(part / kParts, n / kMine * kParts + part % kParts);
    };
    // Step i of a stage: key i * kKeysAtOnce + my_key of this warp's, piece my_piece. (Eight codes of a piece become 16 bytes and go to every second place of a
    // 128-byte row: eight lanes store to all of the banks if they have four pieces of two keys.)
    constexpr bool kInterleave = FP8 && kPieces == 8;
    const int my_key = kInterleave ? ((lane >> 2) & 1) | (lane >> 4 << 1) : lane / kPieces;
    const int my_piece = kInterleave ? (lane & 3) | ((lane >> 3) & 1) << 2 : lane % kPieces;
    auto address = [&](const uint8_t* mine, int i) {
      return reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), i * kKeysAtOnce + my_key)) + my_piece * 16;
    };
    // where 16 bytes of 16-bit elements go, piece c of the key: 128-byte rows, 128-byte swizzle (the key's low bits are those of i and of my_key, apart)
    auto slot = [&](uint32_t base, int c, int i) {
      return base + (c >> 3) * (kKeys * 128) + my_key * 128 + (((uint32_t)((c & 7) ^ my_key) << 4) ^ (((i * kKeysAtOnce) & 7) << 4)) + i * kKeysAtOnce * 128;
    };
    // Asks for stage n: into its place in the ring, or as codes into this warp's own
    auto request = [&](uint32_t n, uint32_t base) {
      const int part = first_part + n % kMine, kv = part / kParts;
      if (n % kMine == 0) next_tile();
      const uint8_t* mine = from[0];
      if constexpr (!Cfg::kSplit) mine = kv ? from[1] : from[0];
      const int beside = (part % kParts) * Cfg::kWidth * es;
      auto to = [&](int i) { return FP8 ? base + i * 512 + lane * 16 : slot(base, my_piece, i); };
      if (__builtin_expect((absent | unknown) == 0, 1)) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) ptx::cp_async_16(to(i), address(mine, i) + beside, 16u);
      } else {
        const uint8_t* lost = reinterpret_cast<const uint8_t*>(FP8 ? &not_a_number8 : &not_a_number16);
#pragma unroll 1
        for (int i = 0; i < kSteps; ++i) {
          const uint8_t* src = address(mine, i) + beside;
          const int key = i * kKeysAtOnce + my_key;
          const bool none = (absent >> key) & 1u, nan = (unknown >> key) & 1u;
          ptx::cp_async_16(to(i), nan ? lost : none ? static_cast<const uint8_t*>(a.q) : src, none || (nan && kv) ? 0u : 16u);
        }
      }
    };
    if constexpr (!FP8) {
      for (uint32_t n = 0; n % kMine != 0 || w.more(); ++n) {
        const Place to = place(n);
        ok = ptx::mbar_wait(empty_bar(to.at), (to.phase & 1) ^ 1, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) break;
        request(n, sKV + to.at * Cfg::kStage + row0 * 128);
        ptx::cp_async_arrive(full_bar(to.at));  // when they have landed
      }
    } else {
      // Every lane reads back what it has copied itself. (Codes held in registers on their way took so many that few bytes were under way.)
      constexpr uint32_t kAhead = Cfg::kRaw - 1;
      const uint32_t raw = sRaw + (warp - Cfg::kProducerWarp) * Cfg::kRaw * Cfg::kRawStage;
      uint32_t asked = 0;
      for (uint32_t m = 0;; ++m) {
        if (asked % kMine != 0 || w.more()) {
          request(asked, raw + asked % Cfg::kRaw * Cfg::kRawStage);
          ++asked;
        }
        ptx::cp_async_commit();
        if (m < kAhead) continue;
        const uint32_t n = m - kAhead;
        if (n >= asked) break;
        const Place to = place(n);
        ok = ptx::mbar_wait(empty_bar(to.at), (to.phase & 1) ^ 1, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) break;
        ptx::cp_async_wait<kAhead>();
        const uint32_t base = sKV + to.at * Cfg::kStage + row0 * 128, codes = raw + n % Cfg::kRaw * Cfg::kRawStage + lane * 16;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const uint4 v = ptx::ld_shared_16(codes + i * 512);
          uint4 lo, hi;
          widen4(v.x, lo.x, lo.y);
          widen4(v.y, lo.z, lo.w);
          widen4(v.z, hi.x, hi.y);
          widen4(v.w, hi.z, hi.w);
          ptx::st_shared_16(slot(base, 2 * my_piece, i), lo);
          ptx::st_shared_16(slot(base, 2 * my_piece + 1, i), hi);
        }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(full_bar(to.at));
      }
    }
    ptx::cp_async_wait_all();
  } else if (warp >= Cfg::kOutputWarp) {
    ptx::give_registers<Cfg::kOtherRegs, Cfg::kLaunchRegs>();  // the same instruction for the group's four warps
    // ------------------------------------------------------------------ queries ahead of their row tile: two warps
    if (Cfg::kQueryWarps && (warp == Cfg::kQWarp || warp == Cfg::kQWarp + 1)) {
      for (int seg = 0; w.more(); w.next(), ++seg) {
        ok = ptx::mbar_wait(q_empty, (seg & 1) ^ 1, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) break;
        load_queries((warp - Cfg::kQWarp) * 32, 64, seg);
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(q_full);
      }
    }
    // ------------------------------------------------------------------ the products, each issued by a thread of its own: the scores of the next tiles do not
    // wait for the weights of this one
    // Operands come by ordinary stores and small copies of other threads. What orders them before the products is the issuing thread's fence behind its wait:
    // a fence of the threads that bring keys would wait for everything that they have under way (FP8 cache, 64 x 16384: 620 us).
    constexpr int kPRow = NT >= 64 ? 128 : NT * 2;
    if (warp == Cfg::kScoreWarp && ptx::elect_one()) {
      constexpr uint32_t idesc = ptx::idesc_f16_f32(kBf16, 0, 128, Cfg::kSCols);
      uint32_t x = 0, stage = 0;  // tiles and stages of keys so far
      for (int seg = 0; w.more() && ok; w.next(), ++seg) {
        ok = ptx::mbar_wait(q_full, seg & 1, abort_flag);
        for (int t = w.t0; t < w.t1 && ok; ++t, ++x) {
          // the scores that were in this buffer have been read, or the weights that took their place multiplied
          if (x >= 2) ok = ptx::mbar_wait(Cfg::kRowsInLanes ? o_done(x) : p_full(x), ((x >> 1) - 1) & 1, abort_flag);
#pragma unroll
          for (int part = 0; part < kParts && ok; ++part, ++stage) {
            const Place from = place_of(0, stage);
            ok = ptx::mbar_wait(full_bar(from.at), from.phase & 1, abort_flag);
            if (!ok) break;
            ptx::fence_proxy_async_smem();
            ptx::tc_fence_after();
            const ptx::Operand keys = ptx::operand_sw128(sKV + from.at * Cfg::kStage), queries = ptx::operand_sw128(sQ + part * 2 * (NT * 128));
            const uint32_t d = tmem_base + (x & 1) * Cfg::kSCols;
#pragma unroll
            for (int k = 0; k < Cfg::kWidth / 16; ++k) {
              const uint32_t in_row = (k & 3) * 32, block = k >> 2;
              const ptx::Operand kk = keys.at(block * (kKeys * 128) + in_row), qq = queries.at(block * (NT * 128) + in_row);
              if (Cfg::kRowsInLanes) ptx::mma_f16(d, qq, kk, idesc, part > 0 || k > 0);
              else ptx::mma_f16(d, kk, qq, idesc, part > 0 || k > 0);
            }
            ptx::mma_commit(empty_bar(from.at));
          }
          if (ok) ptx::mma_commit(s_full(x));
        }
        if (ok && Cfg::kQueryWarps) ptx::mma_commit(q_empty);
      }
    }
    if (warp == Cfg::kOutputWarp && ptx::elect_one()) {
      constexpr uint32_t idesc = Cfg::kRowsInLanes ? ptx::idesc_f16_f32(kBf16, 2, 128, D) : ptx::idesc_f16_f32(kBf16, 3, 128, NT);
      // heads of 64 fill half of the lanes: the other half repeats them
      constexpr uint32_t kNextV = D == 64 && !Cfg::kRowsInLanes ? 0u : kKeys * 128u;
      uint32_t x = 0, stage = 0;  // tiles and stages of values so far
      for (; w.more() && ok; w.next()) {
        for (int t = w.t0; t < w.t1 && ok; ++t, ++x) {
          const uint32_t own = x & 1;
          ok = ptx::mbar_wait(p_full(own), (x >> 1) & 1, abort_flag);
          const uint32_t o = tmem_base + Cfg::kTmemO + (Cfg::kTurns ? own * Cfg::kOCols : 0);
          const uint32_t before = t - w.t0 > (Cfg::kTurns ? 1 : 0);  // O holds earlier tiles
#pragma unroll
          for (int part = 0; part < kParts && ok; ++part, ++stage) {
            const Place from = place_of(1, stage);
            ok = ptx::mbar_wait(full_bar(from.at), from.phase & 1, abort_flag);
            if (!ok) break;
            ptx::fence_proxy_async_smem();
            ptx::tc_fence_after();
            const ptx::Operand values = ptx::operand_depth_rows<128>(sKV + from.at * Cfg::kStage, kNextV);
            const ptx::Operand weights = ptx::operand_depth_rows<kPRow>(sP + own * Cfg::kPBytes, kKeys * 128);
#pragma unroll
            for (int k = 0; k < kKeys / 16; ++k) {
              if (Cfg::kRowsInLanes)  // each half of the keys into its own O
                ptx::mma_f16_ts(o + (k >> 2) * Cfg::kOCols, tmem_base + own * Cfg::kSCols + (k >> 2) * 64 + (k & 3) * 8, values.at(k * 2048), idesc,
                                before || (k & 3));
              else ptx::mma_f16(o + part * NT, values.at(k * 2048), weights.at(k * 16 * kPRow), idesc, before || k > 0);
            }
            ptx::mma_commit(empty_bar(from.at));
          }
          if (ok) ptx::mma_commit(o_done(own));
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax: two groups of four warps
    // What a warp decided alone would leave the others at a barrier: where a wait may have failed, all threads of a group, or all, decide together.
    ptx::give_registers<Cfg::kSoftmaxRegs, Cfg::kLaunchRegs>();
    const int group = warp >> 2, r = threadIdx.x & 127, bar = 1 + group;
    constexpr int kBoth = kBothGroups;
    constexpr int kStep = Cfg::kTurns ? 2 : 1, kCols = Cfg::kCols;
    const uint32_t lane_base = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t o_own = lane_base + Cfg::kTmemO + (Cfg::kTwoO ? group * Cfg::kOCols : group * kCols);
    SplitRows begun = {0, 0, 0, 0, 0};
    uint32_t g = 0;  // tiles of this CTA so far
    for (int seg = 0; w.more(); w.next(), ++seg) {
      const Seq& s = w.s;
      if constexpr (!Cfg::kQueryWarps) {  // (the last scores of the row tile before have been read)
        load_queries(warp * 32, 256, seg);
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(q_full);
        if (kRowScales) ptx::any_of(kBoth, 256, false);
      }
      const int rows = min(NT, s.n * p.group - w.qt * NT), prefix = s.len - s.n;
      const int first_token = fast_div(w.qt * NT, p.group_div), last_token = fast_div(w.qt * NT + rows - 1, p.group_div);
      const float* scales = row_scale + (seg & 3) * NT;
      float c = p.scale_log2;
      if (FP8 && a.k_scale) c *= ld_operand(a.k_scale + (a.k_scales > 1 ? w.h : 0));
      const bool whole = w.t0 == 0 && w.t1 == s.key_tiles;
      if (!whole && w.t0 == 0) begun = {s.start, w.qt, w.h, s.n * p.group, 1 + (int)((s.units(kExtraTiles<NT>) - w.end + line[2] - 1) / line[2])};
      const int64_t slot0 = (2 * (int64_t)blockIdx.x + (w.t0 == 0 ? 1 : 0)) * p.row_slots;
      const float v_scale = FP8 && a.v_scale ? ld_operand(a.v_scale + (a.v_scales > 1 ? w.h : 0)) : 1.f;
      const int mine = w.t0 + (Cfg::kTurns ? (int)((g ^ (uint32_t)group) & 1) : 0);  // this group's first tile
      bool odd_values = false;  // this thread met a value that is not finite among the sequence's own

      // Before the values of tile t are multiplied. Their product with a weight of zero would be NaN where a value is not finite. Those before the sequence's own
      // tokens every row sees; of its own, which some rows do not, such elements are taken out here and added where they are seen, at the end.
      auto check_values = [&](int t) {
        const int j = t * kKeys + r;
        const uint32_t x = g + (t - w.t0);
        if (!Cfg::kTurns && group != 0) return;  // one group looks at a tile
#pragma unroll 1
        for (int part = 0; part < kParts; ++part) {
          const Place from = place_of(1, kParts * x + part);
          ok = ok && ptx::mbar_wait(full_bar(from.at), from.phase & 1, abort_flag);
          if (!ok || j < prefix || j >= s.len) continue;
#pragma unroll 4
          for (int c8 = 0; c8 < Cfg::kWidth / 8; ++c8) {
            const uint32_t at = sKV + from.at * Cfg::kStage + (c8 >> 3) * (kKeys * 128) + r * 128 + (((c8 & 7) ^ (r & 7)) << 4);
            uint4 v = ptx::ld_shared_16(at);
            uint32_t word[4] = {v.x, v.y, v.z, v.w}, odd = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool low = (word[i] & kExponent) == kExponent, high = (word[i] >> 16 & kExponent) == kExponent;
              odd |= low || high;
              word[i] &= (low ? 0xffff0000u : 0xffffffffu) & (high ? 0xffffu : 0xffffffffu);
            }
            if (odd) {
              odd_values = true;
              ptx::st_shared_16(at, make_uint4(word[0], word[1], word[2], word[3]));
            }
          }
        }
      };
      // Bit i of byte loads: does token first + i see this thread's key j, one of the sequence's own or behind its last
      auto seen_by = [&](int j, int first, int count) {
        uint64_t seen = 0;
        const int at = j - prefix;
        const bool known = at >= 0 && j < s.len && (!a.mask || at < a.mask_width);
        const uint8_t* column = static_cast<const uint8_t*>(a.mask) + (int64_t)(s.start + first) * a.mask_ld + at;
        for (int i0 = 0; i0 < count; i0 += 8) {
          uint32_t bit[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {  // (a load behind a branch would be waited for before the next)
            const bool here = known && i0 + i < count;
            bit[i] = a.mask ? (ptx::ld_byte(here ? column + (i0 + i) * a.mask_ld : static_cast<const uint8_t*>(a.q)) != 0 && here)
                            : here && at <= first + i0 + i;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) seen |= (uint64_t)bit[i] << (i0 + i);
        }
        return seen;
      };

      auto wait_for_output = [&] {  // the products with this segment's last tiles
        const uint32_t last = g + (w.t1 - w.t0) - 1;
        if (last >= 1 && w.t1 - w.t0 > 1) ok = ok && ptx::mbar_wait(o_done(last - 1), ((last - 1) >> 1) & 1, abort_flag);
        ok = ok && ptx::mbar_wait(o_done(last), (last >> 1) & 1, abort_flag);
      };

      if constexpr (!Cfg::kRowsInLanes) {
        float* const refs = minus_ref + group * kCols;  // of this group's references, negated
        float* const factors = factor + group * kCols;
        float* const warps = by_warp + group * 4 * kCols;
        int* const tokens = token_of + group * kCols;
        const int n0 = Cfg::kTurns ? 0 : group * kCols;  // this group's first row
        float l[kCols];
#pragma unroll
        for (int i = 0; i < kCols; ++i) l[i] = 0.f;
        if (r < kCols) {
          refs[r] = kNoRef;
          tokens[r] = fast_div(w.qt * NT + n0 + r, p.group_div);
        }
        ptx::any_of(bar, 128, false);
        for (int t = mine; t < w.t1; t += kStep) {
          const uint32_t x_tile = g + (t - w.t0), own = x_tile & 1, phase = x_tile >> 1;
          const uint32_t s_own = lane_base + own * Cfg::kSCols + n0;
          ok = ok && ptx::mbar_wait(s_full(own), phase & 1, abort_flag);
          ptx::tc_fence_after();
          const int j = t * kKeys + r;  // this thread's key
          // the tile's keys that not every row sees
          const bool masked = t * kKeys + kKeys > (a.mask ? prefix : prefix + first_token + 1);
          uint64_t seen = 0;
          if (__builtin_expect(masked, 0)) {
            seen = seen_by(j, first_token, last_token - first_token + 1);
            if (s.n > 1 || a.mask) check_values(t);
          }
          float x[kCols];  // exponents of this thread's key and this group's rows, without their reference
          {
            uint32_t v[32];
            if constexpr (kCols == 16) {
              ptx::tmem_ld16(s_own, v);
              ptx::tmem_ld_wait16(v);
            } else {
              ptx::tmem_ld32(s_own, v);
              ptx::tmem_ld_wait(v);
            }
#pragma unroll
            for (int i = 0; i < kCols; i += 4) {
              float4 by = make_float4(c, c, c, c);
              if constexpr (kRowScales) {
                by = ld_shared_f4(scales + n0 + i);
                by.x *= c, by.y *= c, by.z *= c, by.w *= c;
              }
              x[i] = __uint_as_float(v[i]) * by.x, x[i + 1] = __uint_as_float(v[i + 1]) * by.y;
              x[i + 2] = __uint_as_float(v[i + 2]) * by.z, x[i + 3] = __uint_as_float(v[i + 3]) * by.w;
            }
          }
          if (__builtin_expect(masked && j >= prefix, 0)) {
#pragma unroll
            for (int i = 0; i < kCols; i += 4) {
              const int4 token = *reinterpret_cast<const int4*>(tokens + i);
              if (!((seen >> (token.x - first_token)) & 1)) x[i] = -INFINITY;
              if (!((seen >> (token.y - first_token)) & 1)) x[i + 1] = -INFINITY;
              if (!((seen >> (token.z - first_token)) & 1)) x[i + 2] = -INFINITY;
              if (!((seen >> (token.w - first_token)) & 1)) x[i + 3] = -INFINITY;
            }
          }
          float above[2] = {-INFINITY, -INFINITY};  // largest of them over its reference
#pragma unroll
          for (int i = 0; i < kCols; i += 4) {
            const float4 m = ld_shared_f4(refs + i);
            above[0] = ptx::max3(above[0], x[i] + m.x, x[i + 1] + m.y);
            above[1] = ptx::max3(above[1], x[i + 2] + m.z, x[i + 3] + m.w);
          }
          // the product that read this buffer of P^T is complete (with tiles in turn it is the last one that this group's O was in)
          if (x_tile >= 2) ok = ok && ptx::mbar_wait(o_done(own), (phase - 1) & 1, abort_flag);
          if (__builtin_expect(ptx::any_of(bar, 128, fmaxf(above[0], above[1]) > kReach<M> || t == mine || !ok), 0)) {
            // Rows whose largest score lies too far above their reference take it as the new one
            const bool moves = t > mine;
            if (moves && !Cfg::kTurns) ok = ok && ptx::mbar_wait(o_done(own ^ 1), ((x_tile - 1) >> 1) & 1, abort_flag);
            if (ptx::any_of(bar, 128, !ok)) {
              ok = false;
              break;
            }
            const float of_lane = across_lanes(x, [](float x, float y) { return fmaxf(x, y); });
            if (lane < kCols) warps[(warp & 3) * kCols + lane] = of_lane;
            ptx::any_of(bar, 128, false);
            if (r < kCols) {
              const float top = fmaxf(fmaxf(warps[r], warps[kCols + r]), fmaxf(warps[2 * kCols + r], warps[3 * kCols + r])), old = -refs[r];
              const bool move = top > old + kReach<M>;
              const float next = top - kBelow<M>;
              factors[r] = move ? ptx::ex2(old - next) : 1.f;
              if (move) refs[r] = -next;
            }
            ptx::any_of(bar, 128, false);
            if (moves) {
#pragma unroll
              for (int i = 0; i < kCols; i += 4) {
                const float4 f = ld_shared_f4(factors + i);
                l[i] *= f.x, l[i + 1] *= f.y, l[i + 2] *= f.z, l[i + 3] *= f.w;
              }
              ptx::tc_fence_after();
#pragma unroll 1
              for (int d = 0; d < kParts * kCols; d += 16) {
                const int part = d / kCols, n = d - part * kCols;
                uint32_t o[32], scaled[16];
                ptx::tmem_ld16(o_own + part * NT + n, o);
                ptx::tmem_ld_wait16(o);
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                  const float4 f = ld_shared_f4(factors + n + i);
                  scaled[i] = __float_as_uint(__uint_as_float(o[i]) * f.x), scaled[i + 1] = __float_as_uint(__uint_as_float(o[i + 1]) * f.y);
                  scaled[i + 2] = __float_as_uint(__uint_as_float(o[i + 2]) * f.z), scaled[i + 3] = __float_as_uint(__uint_as_float(o[i + 3]) * f.w);
                }
                ptx::tmem_st16(o_own + part * NT + n, scaled);
              }
              ptx::tmem_st_wait();
            }
          }
          constexpr int kRow = NT >= 64 ? 128 : NT * 2;  // bytes of a key's row of P^T
          const int swizzle = kRow == 128 ? r & 7 : kRow == 64 ? (r >> 1) & 3 : (r >> 2) & 1;
          const uint32_t row = sP + own * Cfg::kPBytes + r * kRow;
#pragma unroll
          for (int i = 0; i < kCols; i += 8) {
            uint32_t out[4];
            const float4 m0 = ld_shared_f4(refs + i), m1 = ld_shared_f4(refs + i + 4);
            ptx::add_two(x[i], x[i + 1], m0.x, m0.y);
            ptx::add_two(x[i + 2], x[i + 3], m0.z, m0.w);
            ptx::add_two(x[i + 4], x[i + 5], m1.x, m1.y);
            ptx::add_two(x[i + 6], x[i + 7], m1.z, m1.w);
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const float e0 = ptx::ex2(x[i + e]), e1 = ptx::ex2(x[i + e + 1]);
              ptx::add_two(l[i + e], l[i + e + 1], e0, e1);
              out[e / 2] = pack2<M>(e0, e1);
            }
            ptx::st_shared_16(row + ((((n0 + i) / 8) ^ swizzle) << 4), make_uint4(out[0], out[1], out[2], out[3]));
          }
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(p_full(own));
        }
        // sums of the weights: over this warp's keys, then over the warps
        const float of_lane = across_lanes(l, [](float x, float y) { return x + y; });
        if (lane < kCols) warps[(warp & 3) * kCols + lane] = of_lane;
        wait_for_output();
        if (ptx::any_of(kBoth, 256, !ok)) break;
        ptx::tc_fence_after();
        if (threadIdx.x < NT) {  // with tiles in turn, both groups' sums on the larger reference
          const int n = threadIdx.x, at = w.qt * NT + n, token = fast_div(at, p.group_div);
          const float* b = by_warp + (Cfg::kTurns ? n : n / kCols * 4 * kCols + n % kCols);
          const float sum0 = (b[0] + b[kCols]) + (b[2 * kCols] + b[3 * kCols]), ref0 = -minus_ref[n];
          float sum1 = 0.f, ref1 = ref0;
          if constexpr (Cfg::kTurns) sum1 = (b[4 * NT] + b[5 * NT]) + (b[6 * NT] + b[7 * NT]), ref1 = -minus_ref[NT + n];
          const float ref = fmaxf(ref0, ref1);
          const float f0 = sum0 == 0.f ? 0.f : ptx::ex2(ref0 - ref), f1 = sum1 == 0.f ? 0.f : ptx::ex2(ref1 - ref);
          const float sum = sum0 * f0 + sum1 * f1, by = whole ? (sum == 0.f ? 0.f : v_scale / sum) : 1.f;
          factor[n] = sum0 == 0.f ? kNothing : f0 * by;
          factor[NT + n] = sum1 == 0.f ? kNothing : f1 * by;
          out_row[n] = (s.start + token) * a.q_heads + w.h * p.group + at - token * p.group;
          if (n < rows) {
            if (!whole) p.part_ml[slot0 + n] = make_float2(ref, sum);
            else if (a.lse) a.lse[out_row[n]] = sum == 0.f ? -INFINITY : (ref + log2f(sum)) * 0.6931471805599453f;
          }
        }
        ptx::any_of(kBoth, 256, false);
        if (r < Cfg::kWidth) {
#pragma unroll 1
          for (int d0 = group * 16; d0 < kParts * NT; d0 += 32) {  // the groups take every second 16 columns
            const int part = d0 / NT, first = d0 - part * NT, d = part * 128 + r;
            if (first >= rows) continue;  // the same for the whole group
            uint32_t o0[32], o1[32];
            ptx::tmem_ld16(lane_base + Cfg::kTmemO + d0, o0);
            if constexpr (Cfg::kTwoO) ptx::tmem_ld16(lane_base + Cfg::kTmemO + Cfg::kOCols + d0, o1);
            ptx::tmem_ld_wait16(o0);
            if constexpr (Cfg::kTwoO) ptx::tmem_ld_wait16(o1);
            T* const out = static_cast<T*>(a.out) + d;
            float* const partial = p.part_o + (slot0 + first) * D + d;
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const float4 f0 = ld_shared_f4(factor + first + i), f1 = ld_shared_f4(factor + NT + first + i);
              const int4 to = *reinterpret_cast<const int4*>(out_row + first + i);
              // a group that has seen nothing of a row adds nothing, whatever its O holds; one whose weights vanish beside the other's still adds a NaN
              auto both = [&](int e, float y0, float y1) {
                float sum = y0 == kNothing ? 0.f : __uint_as_float(o0[e]) * y0;
                if constexpr (Cfg::kTwoO) sum += y1 == kNothing ? 0.f : __uint_as_float(o1[e]) * y1;
                return sum;
              };
              const float x[4] = {both(i, f0.x, f1.x), both(i + 1, f0.y, f1.y), both(i + 2, f0.z, f1.z), both(i + 3, f0.w, f1.w)};
              const int rows_to[4] = {to.x, to.y, to.z, to.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (first + i + e >= rows) continue;
                if (whole) out[(int64_t)rows_to[e] * D] = from_f32<T>(x[e]);
                else partial[(i + e) * D] = x[e];
              }
            }
          }
        }
      } else {
        // A thread per row, 64 keys of a tile in its registers: reference and sum are its own
        const bool busy = (warp & 3) * 32 < rows;  // the same for the whole warp
        const int at = w.qt * NT + min(r, rows - 1), token = fast_div(at, p.group_div);
        const int64_t to = (int64_t)(s.start + token) * a.q_heads + w.h * p.group + at - token * p.group;
        float m = -kNoRef, l = 0.f, scale = c;
        for (int t = mine; t < w.t1; ++t) {
          const uint32_t x_tile = g + (t - w.t0), own = x_tile & 1, phase = x_tile >> 1;
          const uint32_t s_own = lane_base + own * Cfg::kSCols + group * 64;
          ok = ok && ptx::mbar_wait(s_full(own), phase & 1, abort_flag);
          ptx::tc_fence_after();
          if (t == mine) {
            if (kRowScales) scale = c * scales[min(r, rows - 1)];
            if (FP8 && scale == 0.f) scale = FLT_MIN;  // an underflow would make NaN of keys that are not seen, -infinity here already
          }
          const bool masked = t * kKeys + kKeys > (a.mask ? prefix : prefix + first_token + 1);
          // Every second tile has the same words: a warp may be at the next masked tile while the others still read those of this one, and it is past that
          // tile's barrier, which they reach with them read, before it writes these again
          uint32_t* const words = seen_words + (own * 2 + group) * NT * 4;
          if (__builtin_expect(masked, 0)) {  // thread r finds out who sees key r; a word per token and 32 keys. (Each group for itself: they need not be at the same tile.)
            const int j = t * kKeys + r;
            for (int i0 = 0; i0 <= last_token - first_token; i0 += 64) {
              const int count = min(64, last_token - first_token + 1 - i0);
              const uint64_t seen = seen_by(j, first_token + i0, count);
              for (int i = 0; i < count; ++i) {
                const uint32_t word = __ballot_sync(0xffffffffu, j < prefix || ((seen >> i) & 1));
                if (lane == 0) words[(i0 + i) * 4 + (warp & 3)] = word;
              }
            }
            if (s.n > 1 || a.mask) check_values(t);
            ptx::any_of(bar, 128, false);
          }
          if (busy) {
            uint32_t v[2][32];
#pragma unroll
            for (int i = 0; i < 2; ++i) ptx::tmem_ld32(s_own + i * 32, v[i]);
#pragma unroll
            for (int i = 0; i < 2; ++i) ptx::tmem_ld_wait(v[i]);
            if (__builtin_expect(masked, 0)) {
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const uint32_t word = words[(token - first_token) * 4 + group * 2 + q];
#pragma unroll
                for (int i = 0; i < 32; ++i) v[q][i] = (word >> i) & 1u ? v[q][i] : 0xff800000u;
              }
            }
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int i = 0; i < 32; i += 2) top[(i >> 1) & 3] = ptx::max3(top[(i >> 1) & 3], __uint_as_float(v[q][i]), __uint_as_float(v[q][i + 1]));
            const float largest = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
            const bool move = largest > m + kReach<M>;
            const float next = largest - kBelow<M>;
            if (t == mine) {
              if (move) m = next;
            } else if (__builtin_expect(__any_sync(0xffffffffu, move), 0)) {
              const float f = move ? ptx::ex2(m - next) : 1.f;
              if (move) m = next;
              l *= f;
              // (not for a phase two ahead: the scores of the tile before were asked for behind the product before this one)
              ok = ok && ptx::mbar_wait(o_done(own ^ 1), ((x_tile - 1) >> 1) & 1, abort_flag);
              ptx::tc_fence_after();
#pragma unroll 1
              for (int d = 0; d < D; d += 16) {
                uint32_t o[32], scaled[16];
                ptx::tmem_ld16(o_own + d, o);
                ptx::tmem_ld_wait16(o);
#pragma unroll
                for (int i = 0; i < 16; ++i) scaled[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                ptx::tmem_st16(o_own + d, scaled);
              }
            }
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t out[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float e0, e1;
                ptx::fma_two(e0, e1, __uint_as_float(v[q][2 * i]), __uint_as_float(v[q][2 * i + 1]), scale, scale, -m, -m);
                e0 = ptx::ex2(e0), e1 = ptx::ex2(e1);
                ptx::add_two(sum[(i & 1) * 2], sum[(i & 1) * 2 + 1], e0, e1);
                out[i] = pack2<M>(e0, e1);
              }
              ptx::tmem_st16(s_own + q * 16, out);  // over scores that are in registers
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            ptx::tmem_st_wait();
          }
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(p_full(own));
        }
        wait_for_output();
        minus_ref[group * NT + r] = m;
        by_warp[group * NT + r] = l;
        if (ptx::any_of(kBoth, 256, !ok)) break;
        ptx::tc_fence_after();
        if (busy) {
          const float ref0 = minus_ref[r], ref1 = minus_ref[NT + r], ref = fmaxf(ref0, ref1), sum0 = by_warp[r], sum1 = by_warp[NT + r];
          float f0 = sum0 == 0.f ? 0.f : ptx::ex2(ref0 - ref), f1 = sum1 == 0.f ? 0.f : ptx::ex2(ref1 - ref);
          const float sum = sum0 * f0 + sum1 * f1;
          if (group == 0 && r < rows) {
            if (!whole) p.part_ml[slot0 + r] = make_float2(ref, sum);
            else if (a.lse) a.lse[to] = sum == 0.f ? -INFINITY : (ref + log2f(sum)) * 0.6931471805599453f;
          }
          const float by = whole ? (sum == 0.f ? 0.f : v_scale / sum) : 1.f;
          f0 *= by, f1 *= by;
          T* const out = static_cast<T*>(a.out) + to * D;
          float* const partial = p.part_o + slot0 * D + r * 4;  // [D / 4][rows][4]: the lanes of a warp store side by side
#pragma unroll 1
          for (int d = group * (D / 2); d < (group + 1) * (D / 2); d += 16) {  // half of the row each
            uint32_t o0[32], o1[32];
            ptx::tmem_ld16(lane_base + Cfg::kTmemO + d, o0);
            ptx::tmem_ld16(lane_base + Cfg::kTmemO + Cfg::kOCols + d, o1);
            ptx::tmem_ld_wait16(o0);
            ptx::tmem_ld_wait16(o1);
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)  // a group that has seen nothing of the row adds nothing, whatever its O holds; a NaN of vanishing weight counts
              x[i] = (sum0 == 0.f ? 0.f : __uint_as_float(o0[i]) * f0) + (sum1 == 0.f ? 0.f : __uint_as_float(o1[i]) * f1);
            if (r < rows) {
              if (whole) {
#pragma unroll
                for (int i = 0; i < 16; i += 8)
                  *reinterpret_cast<uint4*>(out + d + i) =
                      make_uint4(pack2<T>(x[i], x[i + 1]), pack2<T>(x[i + 2], x[i + 3]), pack2<T>(x[i + 4], x[i + 5]), pack2<T>(x[i + 6], x[i + 7]));
              } else {
#pragma unroll
                for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(partial + (d + i) * p.row_slots) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
              }
            }
          }
        }
      }
      ptx::tc_fence_before();
      // (the barrier also says that this segment's tables have been read)
      if (__builtin_expect(ptx::any_of(kBoth, 256, odd_values), 0)) {
        add_odd_values<T, D, NT, FP8>(p, {w.b, w.h, w.qt, s.start, rows, prefix, max(max(prefix, 0), w.t0 * kKeys), min(s.len, w.t1 * kKeys), whole, slot0},
                                      reinterpret_cast<uint32_t*>(factor));
        ptx::any_of(kBoth, 256, false);
      }
      g += w.t1 - w.t0;
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
  if (warp == Cfg::kOutputWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

// Rows whose keys were cut: adds up their pieces, in the order of the line. Every block reads the list of cut tiles and takes its share of their rows: eight at a
// time, a warp each, or where a tile was cut into many pieces one at a time, each warp with some of them.
constexpr int kManyParts = 8, kJoinBlocks = 740;  // (five to an SM)
template <typename T, int D, int NT, bool FP8>
__global__ void __launch_bounds__(256) tree_attention_join_kernel(const __grid_constant__ AttnParams p, int ctas) {
  const b200_tree_attention_args& a = p.a;
  constexpr int kPer = D / 32;  // elements per lane
  __shared__ int ends[256];     // units of work up to each CTA's tile
  __shared__ SplitRows list[256];
  __shared__ int warp_sum[8];
  __shared__ float part_acc[8][D], part_m[8], part_sum[8];
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto rows_of = [&](const SplitRows& t) { return min(NT, t.rows - t.qt * NT); };
  {
    int units = 0;
    if ((int)threadIdx.x < ctas) {
      const int32_t* from = reinterpret_cast<const int32_t*>(p.split + threadIdx.x);
      const SplitRows t = {ld_operand(from), ld_operand(from + 1), ld_operand(from + 2), ld_operand(from + 3), ld_operand(from + 4)};
      list[threadIdx.x] = t;
      units = t.parts == 0 ? 0 : t.parts > kManyParts ? rows_of(t) : (rows_of(t) + 7) / 8;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, units, o);
      if (lane >= o) units += other;
    }
    if (lane == 31) warp_sum[warp] = units;
    __syncthreads();
    for (int i = 0; i < warp; ++i) units += warp_sum[i];
    ends[threadIdx.x] = units;
    __syncthreads();
  }
  const int total = ends[255];
  for (int unit = blockIdx.x; unit < total; unit += gridDim.x) {
    int cta = 0;  // the first whose end lies behind the unit
    for (int step = 128; step > 0; step >>= 1)
      if (ends[cta + step - 1] <= unit) cta += step;
    const int index = unit - (cta ? ends[cta - 1] : 0);
    const SplitRows tile = list[cta];
    const int parts = tile.parts;
    const bool many = parts > kManyParts;
    const int r = many ? index : index * 8 + warp;
    const bool here = r < rows_of(tile);
    const int step = many ? 8 : 1, begin = many ? warp : 0;  // pieces begin, begin + step, ..
    auto slot_of = [&](int i) { return (2 * (int64_t)(cta + i) + (i == 0 ? 1 : 0)) * p.row_slots + r; };
    float m = -kNoRef, sum = 0.f, acc[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
    const int mine = here && begin < parts ? (parts - begin + step - 1) / step : 0;
    for (int i0 = 0; i0 < mine; i0 += 32) {
      float ref = -kNoRef, l = 0.f;
      if (i0 + lane < mine) {
        const float* ml = reinterpret_cast<const float*>(p.part_ml + slot_of(begin + (i0 + lane) * step));
        ref = ld_operand(ml);
        l = ld_operand(ml + 1);
      }
      float top = fmaxf(ref, m);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float old = ptx::ex2(m - top), weight = ptx::ex2(ref - top);
      m = top;
      sum = fmaf(sum, old, l * weight);
#pragma unroll
      for (int k = 0; k < kPer; ++k) acc[k] *= old;
      const int n = min(32, mine - i0);
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const float f = __shfl_sync(0xffffffffu, weight, i);
        const int64_t slot = slot_of(begin + (i0 + i) * step);
        float x[kPer];
        constexpr bool kRowsInLanes = AttnCfg<D, NT, FP8>::kRowsInLanes;
        const float* src = p.part_o + (kRowsInLanes ? (slot - r) * D + (lane * kPer / 4 * p.row_slots + r) * 4 + lane * kPer % 4 : slot * D + lane * kPer);
        if constexpr (kPer == 2) {
          x[0] = ld_operand(src), x[1] = ld_operand(src + 1);
        } else {
#pragma unroll
          for (int k = 0; k < kPer; k += 4) {
            const float4 v = ld_operand(reinterpret_cast<const float4*>(src + k));
            x[k] = v.x, x[k + 1] = v.y, x[k + 2] = v.z, x[k + 3] = v.w;
          }
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k) acc[k] = fmaf(x[k], f, acc[k]);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (many) {  // over the warps
#pragma unroll
      for (int k = 0; k < kPer; ++k) part_acc[warp][lane * kPer + k] = acc[k];
      if (lane == 0) part_m[warp] = m, part_sum[warp] = sum;
      __syncthreads();
      if (warp == 0) {
        for (int i = 1; i < 8; ++i) m = fmaxf(m, part_m[i]);
        sum = 0.f;
#pragma unroll
        for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
        for (int i = 0; i < 8; ++i) {
          const float f = ptx::ex2(part_m[i] - m);
          sum = fmaf(part_sum[i], f, sum);
#pragma unroll
          for (int k = 0; k < kPer; ++k) acc[k] = fmaf(part_acc[i][lane * kPer + k], f, acc[k]);
        }
      }
    }
    if (here && (!many || warp == 0)) {
      const int row = tile.qt * NT + r, token = fast_div(row, p.group_div), head = tile.head * p.group + row - token * p.group;
      const int64_t to = (int64_t)(tile.token + token) * a.q_heads + head;
      const float inv = sum == 0.f ? 0.f : (FP8 && a.v_scale ? ld_operand(a.v_scale + (a.v_scales > 1 ? tile.head : 0)) : 1.f) / sum;
      T* dst = static_cast<T*>(a.out) + to * D + lane * kPer;
#pragma unroll
      for (int k = 0; k < kPer; k += 2) *reinterpret_cast<uint32_t*>(dst + k) = pack2<T>(acc[k] * inv, acc[k + 1] * inv);
      if (a.lse && lane == 0) a.lse[to] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
    }
    if (many) __syncthreads();  // the tables have been read
  }
}

// Rows of a tile: those of one sequence's new tokens, as far as the host knows their number (the mask's width, else their mean).
inline int attention_rows(const b200_tree_attention_args& a) {
  const int64_t n = a.q_starts == nullptr ? 1 : a.mask ? a.mask_width : cdiv(a.tokens, a.sequences);
  const int64_t rows = (n < 1 ? 1 : n) * (a.q_heads / a.kv_heads);
  return rows <= 16 ? 16 : rows <= 32 || a.dim > 128 ? 32 : rows <= 64 ? 64 : 128;  // more rows of 256 leave no room for the ring
}
// CTAs of a call: no more than there can be tiles
inline int64_t attention_grid(const b200_tree_attention_args& a) {
  const int64_t group = a.q_heads / a.kv_heads, row_tiles = cdiv(a.tokens * group, attention_rows(a)) + a.sequences;
  const int64_t capacity = a.max_pages * a.page_size, key_tiles = capacity > 0 ? cdiv(capacity, kKeys) : 1;
  const double tiles = (double)row_tiles * a.kv_heads * key_tiles;
  const int sms = sm_count() < 256 ? sm_count() : 256;  // (as many as the joining kernel has threads)
  return tiles < sms ? (int64_t)tiles : sms;
}
inline int attention_row_slots(const b200_tree_attention_args& a) {
  const int64_t rows = a.tokens * (a.q_heads / a.kv_heads), tile = attention_rows(a);
  return (int)(rows < tile ? rows : tile);
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

template <typename T, int D, int NT, bool FP8>
static int launch_attention(const AttnParams& p, int grid, cudaStream_t st) {
  using Cfg = AttnCfg<D, NT, FP8>;
  auto k = tree_attention_kernel<T, D, NT, FP8>;
  if (int rc = allow_smem(k, Cfg::kSmemBytes, "tree_attention_kernel")) return rc;
  // The kernel lets the join go by its end alone: blocks of the join that came as soon as the last copies had landed cost more than their start (131072 keys,
  // cache in L2: 256 rows 51 -> 38 us, 128 rows of one tile 57 -> 30; calls that split little the same)
  if (int rc = launch_dependent(k, dim3((unsigned)grid), Cfg::kThreads, Cfg::kSmemBytes, st, 1, "tree_attention", p)) return rc;
  return launch_dependent(tree_attention_join_kernel<T, D, NT, FP8>, dim3(kJoinBlocks), 256, 0, st, 1, "tree_attention", p, grid);
}
template <typename T, int D, int NT>
static int launch_attention(const AttnParams& p, int grid, cudaStream_t st) {
  return p.a.cache_dtype == B200_E4M3 ? launch_attention<T, D, NT, true>(p, grid, st) : launch_attention<T, D, NT, false>(p, grid, st);
}
template <typename T, int D>
static int launch_attention(const AttnParams& p, int grid, cudaStream_t st) {
  switch (attention_rows(p.a)) {
    case 16: return launch_attention<T, D, 16>(p, grid, st);
    case 32: return launch_attention<T, D, 32>(p, grid, st);
    case 64:
      if constexpr (D <= 128) return launch_attention<T, D, 64>(p, grid, st);
      return B200_E_UNSUPPORTED;
    default:
      if constexpr (D <= 128) return launch_attention<T, D, 128>(p, grid, st);
      return B200_E_UNSUPPORTED;
  }
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
  // The distance of one thing to the next that does not exist says nothing
  if (a.tokens == 1) p.a.q_token = 0;
  if (a.q_heads == 1) p.a.q_head = 0;
  if (a.pages <= 1) p.a.k_page = p.a.v_page = 0;
  if (a.page_size == 1) p.a.k_token = p.a.v_token = 0;
  if (a.kv_heads == 1) p.a.k_head = p.a.v_head = 0;
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
