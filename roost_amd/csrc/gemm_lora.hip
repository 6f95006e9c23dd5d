// GemmLora for gfx950: a projection shared by every sequence, with each sequence's own low-rank adapter and an addend on
// top.
//
//   y_t = W x_t + scale_a B_a[:, :rank] (A_a[:rank] x_t) + addend_t,   a = the adapter of row t's sequence (or none)
//
// Launches: ShrinkKernel leaves the low-rank rows u_t = scale_a A_a x_t in the workspace, then the product's kernel adds
// B_a u_t to its own sums before they are stored, so the output is written once. One or two short sequences take a single
// launch (FewRowsKernel). Up to 64 rows, and where their tiles fill one round of the CUs, the wavefronts of a workgroup
// split the inner dimension (ProductKernel: bound by the weight's bytes and by latency); more rows go by tiles (TileKernel:
// bound by the matrix instructions). LaunchAll holds the rules between them, with what was measured on both sides.
//
// Sums are fp32. Low-rank rows are fp32 beside f32 adapters; beside bf16 ones the matrix instructions take them in bf16: rounded
// once under a bf16 output (off by at most 2^-8 of each, as a bf16 tensor between two products would be), in three parts that
// hold all 24 bits under an f32 output.
//
// Operands: everything is moved in 16-byte pieces along the inner dimension (8 bf16, 4 f32 or 16 e4m3), from memory
// straight into LDS (global_load_lds, 8 rows of 128 bytes an instruction), and read from there as fragments: a load of a
// fragment from memory touches 16 or 32 rows at once, which the address unit takes one after another (58 requests an
// instruction were counted), while eight whole 128-byte lines are eight. A matrix-instruction fragment of 16 rows is one
// piece a lane: lane l holds row l % 16, piece l / 16 of a 64-byte run. That is the operand layout of
// v_mfma_f32_16x16x32_bf16 as it stands; for f32 (four v_mfma_f32_16x16x4_f32, one word of the piece each) and e4m3 (two
// v_mfma_f32_16x16x32_fp8_fp8, 8 bytes each) the pieces visit the inner dimension in another order, the same for both
// operands, so the sum is over the same products. Weight rows are the first operand and token rows the second: in the
// result lane l holds token l % 16 and the four consecutive outputs 4 (l / 16) .. + 3. The 32-row fragments of the tiles
// are the same with 32 rows and two pieces.

#include <type_traits>

#include "common.h"
#include "row_steps.h"

namespace {

using namespace roost_dev;

constexpr char kOp[] = "gemm_lora";
constexpr uint32_t kMaxRank = 128;
constexpr uint32_t kCus = 256;  // of an MI355X that is one device; only which tiles are taken depends on it

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

struct E4m3 {
  uint8_t bits;
};
// The same rows multiplied as bf16 (an exact conversion, in registers). The e4m3 matrix instructions cut the products of eight
// neighbouring elements at 2^-13 of the power of two of the largest of the eight, and add the eights in fp32: over 4,096
// products of random codes they are 5e-5 of the result off, bf16's 4e-7. That is far below a bf16 output's rounding (2^-8),
// which takes them for their rate, and far above an f32 output's, which therefore takes this form.
struct E4m3AsBf16 {
  uint8_t bits;
};
template <typename E>
constexpr bool kIsE4m3 = std::is_same_v<E, E4m3> || std::is_same_v<E, E4m3AsBf16>;

// The adapters' type beside rows of type E.
template <typename E>
using LowOf = std::conditional_t<std::is_same_v<E, float>, float, uint16_t>;

struct LoraArgs {
  const void* x;
  const float* x_scale;
  const void* w;
  const float* w_scale;
  const void* a;
  const void* b;
  const float* lora_scale;
  const int32_t* ranks;
  const int32_t* slots;
  const int32_t* cu;
  const void* addend;
  void* y;
  float* u;         // [tokens, max_rank]
  uint16_t* u_bf16;  // the same in bf16 parts that add up to it, `parts` arrays one after another (bf16 adapters)
  uint64_t u_part;   // elements of one
  uint32_t parts;
  uint64_t x_stride, addend_stride, y_stride;  // elements
  uint32_t tokens, batch, in_dim, out_dim, adapters, max_rank;
  uint32_t addend_f32, y_f32;
};

// This wavefront's LDS writes are visible to its own lanes' reads after it, and no access moves across.
__device__ __forceinline__ void WaveSync() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// ---- Which adapter a row has ---------------------------------------------------------------------------------------

constexpr int32_t kNoRow = -2;      // the row belongs to no sequence
constexpr int32_t kNoAdapter = -1;

__device__ __forceinline__ uint32_t RankOf(const LoraArgs& g, int32_t slot) {
  if (slot < 0) return 0;
  if (g.ranks == nullptr) return g.max_rank;
  return static_cast<uint32_t>(min(max(g.ranks[slot], 0), static_cast<int32_t>(g.max_rank)));
}

// A sequence's first row, the next one's and its adapter, as stored.
struct Sequence {
  int32_t from, to, slot;
};
__device__ __forceinline__ Sequence SequenceOf(const LoraArgs& g, uint32_t b) {
  return Sequence{g.cu[b], g.cu[b + 1], g.a != nullptr ? g.slots[b] : kNoAdapter};
}

// slot[i] of each lane's sequence's rows, by whole wavefronts (rows t0 .. t0 + n - 1 of the call are slot[0 ..]): a lane
// writes a short sequence's itself, a long one's are written by its wavefront. The last tile may start part of itself past the
// call's rows: there no row is anyone's, whatever the table says.
__device__ __forceinline__ void PutSlots(const LoraArgs& g, Sequence q, uint32_t t0, uint32_t n, int32_t* slot) {
  constexpr int32_t kShort = 4;
  const int64_t rows = t0 < g.tokens ? min(n, g.tokens - t0) : 0, start = t0;
  const auto lo = static_cast<int32_t>(min(max(q.from - start, int64_t{0}), rows));
  const auto hi = static_cast<int32_t>(min(max(q.to - start, int64_t{0}), rows));
  const int32_t s = q.slot < 0 || static_cast<uint32_t>(q.slot) >= g.adapters ? kNoAdapter : q.slot;
  if (hi - lo <= kShort) {
    for (int32_t t = lo; t < hi; ++t) slot[t] = s;
  }
  for (uint64_t left = __ballot(hi - lo > kShort); left != 0; left &= left - 1) {
    const int l = __builtin_ctzll(left);
    const int32_t from = __builtin_amdgcn_readlane(lo, l), to = __builtin_amdgcn_readlane(hi, l);
    const int32_t its = __builtin_amdgcn_readlane(s, l);
    for (int32_t t = from + static_cast<int32_t>(threadIdx.x % 64); t < to; t += 64) slot[t] = its;
  }
}

// slot[i] for rows t0 .. t0 + n - 1, by the `count` wavefronts from `first` on; a barrier must follow.
__device__ __forceinline__ void FillSlotsBy(const LoraArgs& g, uint32_t t0, uint32_t n, uint32_t first, uint32_t count,
                                            int32_t* slot) {
  const Sequence none = {0, 0, kNoAdapter};
  for (uint32_t b = (threadIdx.x / 64 - first) * 64; b < g.batch; b += 64 * count) {
    const uint32_t its = b + threadIdx.x % 64;
    PutSlots(g, its < g.batch ? SequenceOf(g, its) : none, t0, n, slot);
  }
}
__device__ __forceinline__ void FillSlots(const LoraArgs& g, uint32_t t0, uint32_t n, int32_t* slot) {
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) slot[i] = kNoRow;
  __syncthreads();
  FillSlotsBy(g, t0, n, 0, blockDim.x / 64, slot);
}

// ---- Fragments -------------------------------------------------------------------------------------------------------

// Eight e4m3 elements as eight bf16 (exact: e4m3 has three mantissa bits and a smaller exponent range).
__device__ __forceinline__ bf16x8_t Bf16OfE4m3(uint32_t q0, uint32_t q1) {
  u32x4_t v;
  const uint32_t q[2] = {q0, q1};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(q[i]), false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(q[i]), true);
    v[2 * i] = PackBf16Rne(lo[0], lo[1]);
    v[2 * i + 1] = PackBf16Rne(hi[0], hi[1]);
  }
  return __builtin_bit_cast(bf16x8_t, v);
}

// acc += (16 rows) x (16 rows)^T over the 64 bytes that one piece a lane covers.
template <typename E>
__device__ __forceinline__ f32x4_t Mma16(u32x4_t a, u32x4_t b, f32x4_t acc) {
  if constexpr (std::is_same_v<E, uint16_t>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), acc, 0,
                                                   0, 0);
  } else if constexpr (std::is_same_v<E, float>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), acc, 0, 0, 0);
    }
    return acc;
  } else if constexpr (std::is_same_v<E, E4m3>) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u32x2_t pa = {a[2 * i], a[2 * i + 1]}, pb = {b[2 * i], b[2 * i + 1]};
      acc = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(__builtin_bit_cast(long, pa), __builtin_bit_cast(long, pb), acc, 0, 0,
                                                       0);
    }
    return acc;
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(Bf16OfE4m3(a[2 * i], a[2 * i + 1]), Bf16OfE4m3(b[2 * i], b[2 * i + 1]),
                                                    acc, 0, 0, 0);
    }
    return acc;
  }
}

// The operand of Mma32: one piece, or two (e4m3).
template <typename E>
using FragOf = std::conditional_t<std::is_same_v<E, E4m3>, i32x8_t, u32x4_t>;

// acc += (32 rows) x (32 rows)^T over the 32 bytes that one piece a lane covers, or 64 bytes and two pieces (e4m3): lane l
// holds row l % 32, lanes 0 to 31 one half of the bytes, the others the other.
template <typename E>
__device__ __forceinline__ f32x16_t Mma32(FragOf<E> a, FragOf<E> b, f32x16_t acc) {
  if constexpr (std::is_same_v<E, E4m3>) {
    // Block scales of 2^0 (biased exponent 127).
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, acc, 0, 0, 0, 0x7F7F7F7F, 0, 0x7F7F7F7F);
  } else if constexpr (std::is_same_v<E, uint16_t>) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), acc, 0,
                                                   0, 0);
  } else if constexpr (std::is_same_v<E, float>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i]), __uint_as_float(b[i]), acc, 0, 0, 0);
    }
    return acc;
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(Bf16OfE4m3(a[2 * i], a[2 * i + 1]), Bf16OfE4m3(b[2 * i], b[2 * i + 1]),
                                                    acc, 0, 0, 0);
    }
    return acc;
  }
}

// ---- Copies to LDS -------------------------------------------------------------------------------------------------------
//
// Rows are brought in by 128 bytes of the inner dimension, eight rows an instruction, each row's eight pieces from eight
// neighbouring lanes. Loading the fragments themselves, 16 rows at a time with neighbouring lanes in different rows, costs
// one address cycle a lane instead of one for each four: 30 us instead of 15 for a decode product of 64 x 6,144 over 4,096.

using roost::kStepBytes;

// An address that is the same in every lane, in scalar registers whatever the compiler can prove of it.
__device__ __forceinline__ const unsigned char* Uniform(const unsigned char* p) {
  const auto a = reinterpret_cast<uint64_t>(p);
  const uint64_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a));
  const uint64_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a >> 32));
  return reinterpret_cast<const unsigned char*>(hi << 32 | (lo & 0xFFFFFFFFu));
}

// 16 bytes a lane from memory to LDS: lane l's land at lds + 16 l. No register is written; the caller waits. The copy may read
// M0 one wait state after its write (s_nop), which the compiler does not see to inside an assembly block.
__device__ __forceinline__ void Copy16(const void* base, uint32_t off, uint32_t lds) {
  uint32_t m0;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
               : "=&s"(m0) : "v"(off), "s"(base), "s"(lds) : "memory");
}

__device__ __forceinline__ uint32_t LdsAddress(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const unsigned char*)p));
}

// A wavefront's own rows on their way through LDS: kA rows from one base and kB from another, kStages steps at a time. The
// first rows' steps are kSub times as long as the others' and stand as kSub rows each: first all the rows' first 128 bytes,
// then their second. Piece p of row r lies at p ^ (r % 8), so that the 16 rows of a fragment at one piece are free of bank
// conflicts; the copy writes LDS in lane order, so it is the lanes' source addresses that are permuted. Nothing but this
// wavefront waits for it.
template <int kA, int kB, int kSub, int kStages>
struct RowStream {
  static_assert(kA % (8 * kSub) == 0 && kB % 8 == 0, "eight rows an instruction");
  static constexpr int kCopies = (kA + kB) / 8;
  static constexpr uint32_t kStage = (kA + kB) * kStepBytes, kBytes = kStages * kStage;

  const unsigned char *base_a, *base_b;  // the same in every lane
  uint32_t off_a[kA / 8], off_b[kB / 8];  // of this lane's rows 8 i + lane / 8, from their base
  unsigned char* lds;                     // kBytes
  uint32_t bytes;                         // of a row
  uint32_t piece;                         // this lane's, in its rows

  __device__ __forceinline__ void Copy(uint32_t at, uint32_t stage) const {
    unsigned char* to = lds + stage * kStage;
    const uint32_t to_lds = __builtin_amdgcn_readfirstlane(LdsAddress(to));
    const unsigned char *from_a = Uniform(base_a + at * kSub), *from_b = Uniform(base_b + at);
    if (roost::WholeStep(at, bytes)) {
#pragma unroll
      for (int i = 0; i < kA / 8; ++i) Copy16(from_a, off_a[i], to_lds + 1024 * i);
#pragma unroll
      for (int i = 0; i < kB / 8; ++i) Copy16(from_b, off_b[i], to_lds + 128 * kA + 1024 * i);
      return;
    }
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {  // the last, partial step: pieces past the rows' end are zeros, and no copies
      const bool a = i < kA / 8;
      const uint32_t half = a ? 8 * i / (kA / kSub) : 0;
      if (roost::CopiesPiece(at, half, piece, bytes, a ? kSub : 1)) {
        if (a) {
          Copy16(from_a, off_a[a ? i : 0], to_lds + 1024 * i);
        } else {
          Copy16(from_b, off_b[a ? 0 : i - kA / 8], to_lds + 1024 * i);
        }
      } else {
        *reinterpret_cast<u32x4_t*>(to + 1024 * i + 16 * (threadIdx.x % 64)) = u32x4_t{0, 0, 0, 0};
      }
    }
  }

  // use(stage) for the steps first, first + stride, .. (in bytes) of the rows; it is to have read what it needs of the
  // stage into registers when it returns.
  template <typename U>
  __device__ __forceinline__ void Run(uint32_t first, uint32_t stride, U&& use) const {
    const uint32_t steps = roost::StepsOf(first, stride, bytes), by_count = roost::StepsByCount(first, stride, bytes);
#pragma unroll
    for (uint32_t i = 0; i < kStages; ++i) {
      if (i < steps) Copy(first + i * stride, i);
    }
    uint32_t stage = 0;
#pragma unroll 1
    for (uint32_t i = 0; i < steps; ++i) {
      if (i + kStages <= by_count) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kStages - 1) * kCopies) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      }
      use(lds + stage * kStage, [&] {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (i + kStages < steps) Copy(first + (i + kStages) * stride, stage);
      });
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
  }
};

// The piece of a row in a stage.
__device__ __forceinline__ u32x4_t StagePiece(const unsigned char* stage, uint32_t row, uint32_t piece) {
  return *reinterpret_cast<const u32x4_t*>(stage + row * kStepBytes + 16 * (piece ^ (row % 8)));
}

// ---- The low-rank rows -------------------------------------------------------------------------------------------------

// Rows [from, to) of the sequence with adapter `slot`.
struct RowRange {
  uint32_t from, to;
  int32_t slot;
};

// The `at`-th piece of the batch, where every sequence is cut at the multiples of kRows: at most tokens / kRows + batch of
// them. By the whole workgroup, a lane a sequence: the pieces before each are a prefix sum over the workgroup. Empty past
// the last.
template <int kRows>
__device__ __forceinline__ RowRange PieceOf(const LoraArgs& g, uint32_t at) {
  __shared__ uint32_t sums[16];
  __shared__ RowRange found;
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, waves = blockDim.x / 64;
  if (threadIdx.x == 0) found = RowRange{0, 0, kNoAdapter};
  uint32_t before = 0;
  for (uint32_t first = 0; first < g.batch; first += blockDim.x) {
    const uint32_t b = first + threadIdx.x;
    const Sequence q = SequenceOf(g, min(b, g.batch - 1));
    const auto most = static_cast<int32_t>(g.tokens);
    const auto lo = static_cast<uint32_t>(min(max(q.from, 0), most)), hi = static_cast<uint32_t>(min(max(q.to, 0), most));
    const uint32_t pieces = b < g.batch && hi > lo ? (hi - 1) / kRows - lo / kRows + 1 : 0;
    uint32_t sum = pieces;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t other = __shfl_up(sum, d);
      if (lane >= static_cast<uint32_t>(d)) sum += other;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    uint32_t start = before + sum - pieces;
    for (uint32_t w = 0; w < waves; ++w) {
      if (w < wave) start += sums[w];
      before += sums[w];
    }
    if (at >= start && at < start + pieces) {
      const uint32_t block = lo / kRows + (at - start);
      found = RowRange{max(lo, block * kRows), min(hi, (block + 1) * kRows), q.slot};
    }
    if (at < before) break;
  }
  __syncthreads();
  RowRange r = found;
  if (r.slot < 0 || static_cast<uint32_t>(r.slot) >= g.adapters) r.slot = kNoAdapter;
  return r;
}

// acc += one step of a RowStream's rows: kRows of the input (fewer than 16 kT stand for the others too) times 16 kR of an
// adapter's.
template <typename E, int kT, int kR, int kRows, typename Done>
__device__ __forceinline__ void ShrinkStep(const unsigned char* stage, uint32_t lane, Done&& done, f32x4_t (&acc)[kT][kR]) {
  using Low = LowOf<E>;
  constexpr int kSub = sizeof(Low) / sizeof(E);
  u32x4_t a[2 * kSub][kR], x[2 * kSub][kT];
#pragma unroll
  for (int p = 0; p < 2 * kSub; ++p) {
#pragma unroll
    for (int r = 0; r < kR; ++r) a[p][r] = StagePiece(stage, 16 * kR * (p / 2) + 16 * r + lane % 16, 4 * (p % 2) + lane / 16);
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const uint32_t row = (16 * t + lane % 16) % kRows;
      if constexpr (kSub == 1) {
        x[p][t] = StagePiece(stage, 16 * kR + row, 4 * p + lane / 16);
      } else {
        const uint32_t eighth = 4 * p + lane / 16;  // 8 bytes of the row's 128
        const auto* from = stage + (16 * kR * kSub + row) * kStepBytes + 16 * ((eighth / 2) ^ (row % 8)) + 8 * (eighth % 2);
        const u32x2_t q = *reinterpret_cast<const u32x2_t*>(from);
        x[p][t] = u32x4_t{q[0], q[1], 0, 0};
      }
    }
  }
  done();
#pragma unroll
  for (int p = 0; p < 2 * kSub; ++p) {
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const u32x4_t px = kSub == 1 ? x[p][t] : __builtin_bit_cast(u32x4_t, Bf16OfE4m3(x[p][t][0], x[p][t][1]));
#pragma unroll
      for (int r = 0; r < kR; ++r) acc[t][r] = Mma16<Low>(a[p][r], px, acc[t][r]);
    }
  }
}

// Workgroup (i, j): the i-th piece of the batch (rows of one sequence within kRows = 16 kT), ranks 16 kR j .. + 16 kR - 1.
// The wavefronts take alternate steps of the inner dimension and join their sums through LDS. A step is 128 bytes of the
// rows; e4m3 rows meet twice as many bytes of the adapter's, which stand as two rows each. Bound by the rows' bytes: 15,000
// rows of 4096 channels, rank 64, 33 us (3.7 TB/s); one-token sequences by latency: 61 rows of 24 adapters, rank 32, 5.6 us.
template <typename E, int kT, int kR, int kWaves, int kStages>
__global__ void __launch_bounds__(64 * kWaves) ShrinkKernel(LoraArgs g) {
  using Low = LowOf<E>;
  constexpr int kRows = 16 * kT, kSub = sizeof(Low) / sizeof(E);
  using Stream = RowStream<16 * kR * kSub, kRows, kSub, kStages>;
  static_assert(kWaves * Stream::kBytes >= kWaves * kT * kR * 64 * sizeof(f32x4_t), "the sums fit where the rows were");
  __shared__ __align__(16) unsigned char lds[kWaves * Stream::kBytes];
  const uint32_t r0 = 16 * kR * blockIdx.y;
  const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const RowRange range = PieceOf<kRows>(g, blockIdx.x);
  const int32_t s = __builtin_amdgcn_readfirstlane(range.slot);
  const uint32_t from = __builtin_amdgcn_readfirstlane(range.from), to = __builtin_amdgcn_readfirstlane(range.to);
  const uint32_t rank = __builtin_amdgcn_readfirstlane(RankOf(g, s));
  if (from >= to || r0 >= rank) return;
  Stream rows;
  rows.lds = lds + wave * Stream::kBytes;
  rows.bytes = g.in_dim * sizeof(E);
  rows.piece = roost::PieceOfLane(lane);
  rows.base_b = reinterpret_cast<const unsigned char*>(static_cast<const E*>(g.x) + from * g.x_stride);
  // Rows past the piece's and ranks past the adapter's repeat the last; what they give is not stored.
#pragma unroll
  for (int i = 0; i < kRows / 8; ++i) {
    rows.off_b[i] = min(8 * i + lane / 8, to - 1 - from) * static_cast<uint32_t>(g.x_stride * sizeof(E)) + rows.piece;
  }
  rows.base_a = reinterpret_cast<const unsigned char*>(static_cast<const Low*>(g.a) +
                                                       (static_cast<uint64_t>(s) * g.max_rank + r0) * g.in_dim);
#pragma unroll
  for (int k = 0; k < 2 * kR * kSub; ++k) {
    const uint32_t row = 8 * k + lane / 8, of = row % (16 * kR), half = row / (16 * kR);
    rows.off_a[k] = min(of, rank - 1 - r0) * static_cast<uint32_t>(g.in_dim * sizeof(Low)) + rows.piece + half * kStepBytes;
  }
  f32x4_t acc[kT][kR];
#pragma unroll
  for (int t = 0; t < kT; ++t) {
#pragma unroll
    for (int r = 0; r < kR; ++r) acc[t][r] = f32x4_t{0, 0, 0, 0};
  }
  rows.Run(kStepBytes * wave, kStepBytes * kWaves,
           [&](const unsigned char* stage, auto&& done) { ShrinkStep<E, kT, kR, kRows>(stage, lane, done, acc); });
  auto* part = reinterpret_cast<f32x4_t(*)[kT * kR][64]>(lds);
  __syncthreads();
#pragma unroll
  for (int t = 0; t < kT; ++t) {
#pragma unroll
    for (int r = 0; r < kR; ++r) part[wave][t * kR + r][lane] = acc[t][r];
  }
  __syncthreads();
  for (uint32_t item = threadIdx.x; item < kT * kR * 64; item += 64 * kWaves) {
    const uint32_t tile = item / 64, l = item % 64;
    const uint32_t row = from + 16 * (tile / kR) + l % 16, first = r0 + 16 * (tile % kR) + 4 * (l / 16);
    if (row >= to || first >= rank) continue;
    f32x4_t v = part[0][tile][l];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += part[w][tile][l];
    float scale = g.lora_scale != nullptr ? g.lora_scale[s] : 1.0f;
    if constexpr (kIsE4m3<E>) scale *= g.x_scale[row];
    // max_rank is a multiple of 8: the four are the row's own, those past the adapter's rank unused.
    const uint64_t at = static_cast<uint64_t>(row) * g.max_rank + first;
    v *= scale;
    *reinterpret_cast<f32x4_t*>(g.u + at) = v;
    if constexpr (sizeof(Low) == 2) {
      for (uint32_t p = 0; p < g.parts; ++p) {
        const u32x2_t w = {PackBf16Rne(v[0], v[1]), PackBf16Rne(v[2], v[3])};
        *reinterpret_cast<u32x2_t*>(g.u_bf16 + p * g.u_part + at) = w;
        v -= f32x4_t{Bf16LoToF32(w[0]), Bf16HiToF32(w[0]), Bf16LoToF32(w[1]), Bf16HiToF32(w[1])};
      }
    }
  }
}

// ---- After the product -----------------------------------------------------------------------------------------------------

// Words of a 16-byte piece whose elements from `left` on are zeroed (left may be anything; 0 or less zeroes all).
template <typename Low>
__device__ __forceinline__ u32x4_t First(u32x4_t v, int32_t left) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(Low) == 4) {
      if (i >= left) v[i] = 0;
    } else {
      v[i] = 2 * i + 1 < left ? v[i] : 2 * i < left ? v[i] & 0xFFFFu : 0;
    }
  }
  return v;
}
template <typename Low>
__device__ __forceinline__ float Element(u32x4_t v, int i) {
  if constexpr (sizeof(Low) == 4) {
    return __uint_as_float(v[i]);
  } else {
    return i % 2 ? Bf16HiToF32(v[i / 2]) : Bf16LoToF32(v[i / 2]);
  }
}

// v += B_slot[n .. n + 3, :rank] u_t, element by element; outputs past the last repeat it.
template <typename Low>
__device__ __forceinline__ void AddLowRank(const LoraArgs& g, uint32_t t, uint32_t n, int32_t slot, uint32_t rank, f32x4_t& v) {
  constexpr int kPer = 16 / sizeof(Low);
  const float* u = g.u + static_cast<uint64_t>(t) * g.max_rank;
  const Low* b = static_cast<const Low*>(g.b) + static_cast<uint64_t>(slot) * g.out_dim * g.max_rank;
  const Low* row[4];
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) row[e] = b + static_cast<uint64_t>(min(n + e, g.out_dim - 1)) * g.max_rank;
  constexpr int kAhead = 2;  // pieces requested together
#pragma unroll 1
  for (uint32_t r0 = 0; r0 < rank; r0 += kAhead * kPer) {
    f32x4_t ur[kAhead][kPer / 4];
    u32x4_t br[kAhead][4];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const uint32_t r = r0 + k * kPer, at = r < rank ? r : 0;
#pragma unroll
      for (int i = 0; i < kPer / 4; ++i) ur[k][i] = *reinterpret_cast<const f32x4_t*>(u + at + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) br[k][e] = *reinterpret_cast<const u32x4_t*>(row[e] + at);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const auto left = static_cast<int32_t>(rank) - static_cast<int32_t>(r0 + k * kPer);
#pragma unroll
      for (int i = 0; i < kPer; ++i) ur[k][i / 4][i % 4] = i < left ? ur[k][i / 4][i % 4] : 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u32x4_t q = First<Low>(br[k][e], left);
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[e] = fmaf(ur[k][i / 4][i % 4], Element<Low>(q, i), v[e]);
      }
    }
  }
}

// Consecutive elements of a row at an address that may be aligned to an element only.
typedef uint32_t Bf16x4 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t Bf16x8 __attribute__((ext_vector_type(4), aligned(2)));
typedef float F32x4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ float AddendOne(const LoraArgs& g, uint64_t at) {
  return LoadF(g.addend, g.addend_f32 ? ROOST_DTYPE_F32 : ROOST_DTYPE_BF16, static_cast<int64_t>(at));
}
__device__ __forceinline__ void StoreOne(const LoraArgs& g, uint64_t at, float v) {
  if (g.y_f32) {
    static_cast<float*>(g.y)[at] = v;
  } else {
    static_cast<uint16_t*>(g.y)[at] = static_cast<uint16_t>(PackBf16Rne(v, 0.0f));
  }
}

// Adds the addend and stores outputs n .. n + 3 of row t.
__device__ __forceinline__ void Store(const LoraArgs& g, uint32_t t, uint32_t n, f32x4_t v) {
  const uint64_t at = t * g.y_stride + n, from = t * g.addend_stride + n;
  if (g.out_dim - n >= 4) {
    if (g.addend != nullptr) {
      if (g.addend_f32) {
        v += *reinterpret_cast<const F32x4*>(static_cast<const float*>(g.addend) + from);
      } else {
        const Bf16x4 q = *reinterpret_cast<const Bf16x4*>(static_cast<const uint16_t*>(g.addend) + from);
        v += f32x4_t{Bf16LoToF32(q[0]), Bf16HiToF32(q[0]), Bf16LoToF32(q[1]), Bf16HiToF32(q[1])};
      }
    }
    if (g.y_f32) {
      *reinterpret_cast<F32x4*>(static_cast<float*>(g.y) + at) = v;
    } else {
      *reinterpret_cast<Bf16x4*>(static_cast<uint16_t*>(g.y) + at) = Bf16x4{PackBf16Rne(v[0], v[1]), PackBf16Rne(v[2], v[3])};
    }
    return;
  }
#pragma unroll
  for (uint32_t e = 0; e < 3; ++e) {
    if (e < g.out_dim - n) StoreOne(g, at + e, v[e] + (g.addend != nullptr ? AddendOne(g, from + e) : 0.0f));
  }
}

// The scales of e4m3 rows and weights, on outputs n .. n + 3 of row t.
__device__ __forceinline__ f32x4_t Rescaled(const LoraArgs& g, float x_scale, uint32_t n, f32x4_t v) {
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) v[e] *= x_scale * g.w_scale[min(n + e, g.out_dim - 1)];
  return v;
}

// ---- The product of few rows ---------------------------------------------------------------------------------------------

// A piece of low-rank rows for the adapters' type: fp32 as it is; bf16 rounded to nearest, what that leaves staying in ur
// for the next part.
template <typename Low>
__device__ __forceinline__ u32x4_t NextPart(f32x4_t (&ur)[4 / sizeof(Low)]) {
  u32x4_t pu;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(Low) == 2) {
      pu[i] = PackBf16Rne(ur[i / 2][2 * i % 4], ur[i / 2][2 * i % 4 + 1]);
      ur[i / 2][2 * i % 4] -= Bf16LoToF32(pu[i]);
      ur[i / 2][2 * i % 4 + 1] -= Bf16HiToF32(pu[i]);
    } else {
      pu[i] = __float_as_uint(ur[0][i]);
    }
  }
  return pu;
}

// v[m] += B u for kM 16 x 16 tiles side by side, lane l holding outputs n + 16 m + 4 (l / 16) .. + 3 of the row `token`
// with adapter s (l % 16). The rows of the adapters among the 16 are requested sixteen at a time, before the ranks that say
// how much of them counts are known; each adapter's product is kept by its own rows only.
template <typename Low, int kM>
__device__ __forceinline__ void AddLowRankTiles(const LoraArgs& g, uint32_t token, int32_t s, uint32_t n, uint32_t lane,
                                                f32x4_t (&v)[kM]) {
  constexpr uint32_t kPer = 16 / sizeof(Low);
  constexpr int kTogether = kM == 1 ? 16 : 4;  // adapters whose rows are on their way, kM pieces each
  if (__ballot(s >= 0) == 0) return;
  const uint32_t its_rank = RankOf(g, s);
  int32_t at[16];  // a row of the k-th adapter
  int count = 0;
  uint64_t left = __ballot(lane < 16 && s >= 0);
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    at[k] = left != 0 ? __builtin_ctzll(left) : 0;
    count += left != 0;
    left &= ~__ballot(s == __builtin_amdgcn_readlane(s, at[k]));
  }
  uint32_t out[kM];
#pragma unroll
  for (int m = 0; m < kM; ++m) out[m] = min(n + 16 * m + lane % 16, g.out_dim - 1);
  const float* u = g.u + static_cast<uint64_t>(token) * g.max_rank;
#pragma unroll 1
  for (uint32_t r0 = 0; r0 < g.max_rank; r0 += 4 * kPer) {
    if (r0 > 0 && __ballot(its_rank > r0) == 0) break;
    const uint32_t r = r0 + kPer * (lane / 16), from = r < g.max_rank ? r : 0;
    f32x4_t all[kPer / 4];
#pragma unroll
    for (uint32_t i = 0; i < kPer / 4; ++i) all[i] = *reinterpret_cast<const f32x4_t*>(u + from + 4 * i);
#pragma unroll
    for (int k0 = 0; k0 < 16; k0 += kTogether) {
      if (k0 >= count) break;
      u32x4_t b[kTogether][kM];
#pragma unroll
      for (int k = 0; k < kTogether; ++k) {
        if (k0 + k < count) {
          const auto slot = static_cast<uint64_t>(__builtin_amdgcn_readlane(s, at[k0 + k]));
#pragma unroll
          for (int m = 0; m < kM; ++m) {
            const uint64_t at_row = (slot * g.out_dim + out[m]) * g.max_rank;
            b[k][m] = *reinterpret_cast<const u32x4_t*>(static_cast<const Low*>(g.b) + at_row + from);
          }
        }
      }
      f32x4_t ur[kPer / 4];
#pragma unroll
      for (uint32_t i = 0; i < kPer; ++i) ur[i / 4][i % 4] = r + i < its_rank ? all[i / 4][i % 4] : 0.0f;
      const uint32_t parts = sizeof(Low) == 2 ? g.parts : 1;
#pragma unroll 1
      for (uint32_t part = 0; part < parts; ++part) {
        const u32x4_t pu = NextPart<Low>(ur);
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
          if (k0 + k < count) {
            const auto rest = static_cast<int32_t>(__builtin_amdgcn_readlane(its_rank, at[k0 + k])) - static_cast<int32_t>(r);
            const bool its = s == static_cast<int32_t>(__builtin_amdgcn_readlane(s, at[k0 + k]));
#pragma unroll
            for (int m = 0; m < kM; ++m) {
              const f32x4_t d = Mma16<Low>(First<Low>(b[k][m], rest), pu, f32x4_t{0, 0, 0, 0});
              if (its) v[m] += d;
            }
          }
        }
      }
    }
  }
}

// Bound by the weight's bytes on their way from memory and by the latency of the first of them. 64 rows, 4096 to 6144 channels:
// 14 us for 50 MB of weight (3.6 TB/s) and 32 KB of rows a step and CU out of L2; with the workgroups of an XCD on neighbouring
// tiles, against 21 us with neighbours spread over the XCDs.
//
// A workgroup: 16 kN outputs of 16 kT rows. kWaves wavefronts take alternate steps of the inner dimension; beside them kLow
// others find the rows' adapters and compute their outputs, which has as long a chain of loads (sequence, adapter, rank, its
// rows) as the product but moves little. All join their sums through LDS.
template <typename E, int kN, int kT, int kWaves, int kLow, int kStages>
__global__ void __launch_bounds__(64 * (kWaves + kLow)) ProductKernel(LoraArgs g, uint32_t n_tiles) {
  using Stream = RowStream<16 * kN, 16 * kT, 1, kStages>;
  constexpr int kTiles = kN * kT;
  constexpr int kM = kTiles / kLow;  // tiles of outputs by each wavefront with adapters, of 16 rows
  static_assert(kLow % kT == 0 && kM * kLow == kTiles, "as many for each");
  static_assert(kWaves * Stream::kBytes >= (kWaves + 1) * kTiles * 64 * sizeof(f32x4_t), "the sums fit where the rows were");
  __shared__ __align__(16) unsigned char lds[kWaves * Stream::kBytes];
  __shared__ int32_t slot[kLow][16];
  // Workgroups go to the 8 XCDs in turn; each XCD takes one run of the tiles, so that those next to each other in memory
  // are read through one L2.
  const uint32_t tiles = gridDim.x, xcd = blockIdx.x % 8;
  const uint32_t at = xcd * (tiles / 8) + min(xcd, tiles % 8) + blockIdx.x / 8;
  const uint32_t n0 = 16 * kN * (at % n_tiles), t0 = 16 * kT * (at / n_tiles);
  const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  f32x4_t acc[kN][kT];
#pragma unroll
  for (int n = 0; n < kN; ++n) {
#pragma unroll
    for (int t = 0; t < kT; ++t) acc[n][t] = f32x4_t{0, 0, 0, 0};
  }
  f32x4_t low[kM];
  const uint32_t low_t = (wave - kWaves) % kT, low_n = (wave - kWaves) / kT * kM;
  if (wave >= kWaves) {
    // Each finds its rows' adapters by itself, in a table of its own, so that none waits for another.
    int32_t* mine = slot[wave - kWaves];
    if (lane < 16) mine[lane] = kNoRow;
    WaveSync();
    FillSlotsBy(g, t0 + 16 * low_t, 16, wave, 1, mine);
    WaveSync();
#pragma unroll
    for (int m = 0; m < kM; ++m) low[m] = f32x4_t{0, 0, 0, 0};
    const uint32_t token = min(t0 + 16 * low_t + lane % 16, g.tokens - 1);
    AddLowRankTiles<LowOf<E>, kM>(g, token, mine[lane % 16], n0 + 16 * low_n, lane, low);
  } else if (g.w != nullptr) {
    Stream rows;
    rows.lds = lds + wave * Stream::kBytes;
    rows.bytes = g.in_dim * sizeof(E);
    rows.piece = roost::PieceOfLane(lane);
    rows.base_a = reinterpret_cast<const unsigned char*>(static_cast<const E*>(g.w) + static_cast<uint64_t>(n0) * g.in_dim);
    rows.base_b = reinterpret_cast<const unsigned char*>(static_cast<const E*>(g.x) + t0 * g.x_stride);
    // Rows past the last output or token repeat the last one; what they give is not stored.
#pragma unroll
    for (int i = 0; i < 2 * kN; ++i) rows.off_a[i] = min(8 * i + lane / 8, g.out_dim - 1 - n0) * rows.bytes + rows.piece;
#pragma unroll
    for (int i = 0; i < 2 * kT; ++i) {
      rows.off_b[i] = min(8 * i + lane / 8, g.tokens - 1 - t0) * static_cast<uint32_t>(g.x_stride * sizeof(E)) + rows.piece;
    }
    rows.Run(kStepBytes * wave, kStepBytes * kWaves, [&](const unsigned char* stage, auto&& done) {
      u32x4_t w[2][kN], x[2][kT];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int n = 0; n < kN; ++n) w[p][n] = StagePiece(stage, 16 * n + lane % 16, 4 * p + lane / 16);
#pragma unroll
        for (int t = 0; t < kT; ++t) x[p][t] = StagePiece(stage, 16 * kN + 16 * t + lane % 16, 4 * p + lane / 16);
      }
      done();
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int n = 0; n < kN; ++n) {
#pragma unroll
          for (int t = 0; t < kT; ++t) acc[n][t] = Mma16<E>(w[p][n], x[p][t], acc[n][t]);
        }
      }
    });
  }
  __syncthreads();
  auto* part = reinterpret_cast<f32x4_t(*)[kTiles][64]>(lds);
  if (wave < kWaves) {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
      for (int t = 0; t < kT; ++t) part[wave][n * kT + t][lane] = acc[n][t];
    }
  } else {
#pragma unroll
    for (int m = 0; m < kM; ++m) part[kWaves][(low_n + m) * kT + low_t][lane] = low[m];
  }
  __syncthreads();
  // Lane l of a tile holds outputs 4 (l / 16) .. + 3 of row l % 16.
#pragma unroll 1
  for (uint32_t tile = wave; tile < kTiles; tile += kWaves + kLow) {
    const uint32_t row = 16 * (tile % kT) + lane % 16, n = n0 + 16 * (tile / kT) + 4 * (lane / 16);
    if (slot[tile % kT][lane % 16] == kNoRow || n >= g.out_dim) continue;
    f32x4_t v = part[0][tile][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += part[w][tile][lane];
    if constexpr (kIsE4m3<E>) {
      if (g.w != nullptr) v = Rescaled(g, g.x_scale[t0 + row], n, v);
    }
    Store(g, t0 + row, n, v + part[kWaves][tile][lane]);
  }
}

// ---- One or two short sequences -------------------------------------------------------------------------------------------
//
// A chat's single token waits for nothing but latency, so its low-rank rows are not a launch of their own: every workgroup
// computes them all again for its 16 outputs, by wavefronts beside the product's, from rows that the other workgroups read
// as well. That holds for kFewRows rows and, over all sequences, kFewRanks ranks. Against two launches, one row, rank 16:
// 1024 to 6144 channels 6.7 and 12.7 us, 4096 to 6144 15.7 and 19.7 us, 4096 to 14336 30.5 and 31.6 us, 14336 to 4096 32.5
// and 37.9 us.
constexpr uint32_t kFewRows = 8, kFewRanks = 16;

template <typename E>
__global__ void __launch_bounds__(64 * 12) FewRowsKernel(LoraArgs g) {
  using Low = LowOf<E>;
  constexpr int kWaves = 8, kSide = 4, kSub = sizeof(Low) / sizeof(E);
  constexpr uint32_t kPer = 16 / sizeof(Low);
  using Main = RowStream<16, kFewRows, 1, 2>;
  using Side = RowStream<16 * kSub, kFewRows, kSub, 2>;
  __shared__ __align__(16) unsigned char lds[kWaves * Main::kBytes + kSide * Side::kBytes];
  __shared__ __align__(16) float u[16][kFewRanks];  // [row][rank]
  const uint32_t tiles = gridDim.x, xcd = blockIdx.x % 8;
  const uint32_t n0 = 16 * (xcd * (tiles / 8) + min(xcd, tiles % 8) + blockIdx.x / 8);
  const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t piece = roost::PieceOfLane(lane);
  const uint32_t x_row = min(lane / 8, g.tokens - 1) * static_cast<uint32_t>(g.x_stride * sizeof(E)) + piece;
  const auto* x = static_cast<const unsigned char*>(g.x);

  // Of the last wavefront, which joins the sums, and requested before the rows that it sums: the sequences' adapters, their
  // rows of B (of output n0 + lane % 16), and row t's sequence and scales.
  const uint32_t t = lane % 16;
  int32_t slot[2] = {kNoAdapter, kNoAdapter}, its = kNoRow;
  uint32_t rank[2] = {};
  u32x4_t b[2] = {};
  float scale = 1.0f, x_scale = 1.0f;
  f32x4_t acc[1][1] = {{f32x4_t{0, 0, 0, 0}}};
  if (wave >= kWaves) {
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      if (i < g.batch) slot[i] = g.slots[i];
      if (slot[i] < 0 || static_cast<uint32_t>(slot[i]) >= g.adapters) slot[i] = kNoAdapter;
    }
    Side rows;
    rows.lds = lds + kWaves * Main::kBytes + (wave - kWaves) * Side::kBytes;
    rows.bytes = g.in_dim * sizeof(E);
    rows.piece = piece;
    rows.base_a = static_cast<const unsigned char*>(g.a);
    rows.base_b = x;
    rows.off_b[0] = x_row;
#pragma unroll
    for (int k = 0; k < 2 * kSub; ++k) {
      // Row j: rank j % max_rank of sequence j / max_rank; those of no adapter repeat the first row, and their sums are not
      // kept.
      const uint32_t row = 8 * k + lane / 8, j = row % 16, half = row / 16, i = j / g.max_rank;
      const int32_t its = i == 0 ? slot[0] : i == 1 ? slot[1] : kNoAdapter;
      const uint32_t of = its >= 0 ? static_cast<uint32_t>(its) * g.max_rank + j % g.max_rank : 0;
      rows.off_a[k] = of * static_cast<uint32_t>(g.in_dim * sizeof(Low)) + piece + half * kStepBytes;
    }
    if (wave == kWaves + kSide - 1) {
      const uint32_t out = min(n0 + lane % 16, g.out_dim - 1), j = kPer * (lane / 16);
      if constexpr (kIsE4m3<E>) x_scale = g.x_scale[min(t, g.tokens - 1)];
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) {
        rank[i] = RankOf(g, slot[i]);
        if (i < g.batch && t < g.tokens && static_cast<int32_t>(t) >= g.cu[i] && static_cast<int32_t>(t) < g.cu[i + 1]) {
          its = i;
          scale = g.lora_scale != nullptr && slot[i] >= 0 ? g.lora_scale[slot[i]] : 1.0f;
        }
        if (slot[i] >= 0 && j < kFewRanks && j / g.max_rank == i) {
          const uint64_t row = static_cast<uint64_t>(slot[i]) * g.out_dim + out;
          b[i] = *reinterpret_cast<const u32x4_t*>(static_cast<const Low*>(g.b) + row * g.max_rank + j % g.max_rank);
        }
      }
    }
    if (slot[0] >= 0 || slot[1] >= 0) {
      rows.Run(kStepBytes * (wave - kWaves), kStepBytes * kSide,
               [&](const unsigned char* stage, auto&& done) { ShrinkStep<E, 1, 1, kFewRows>(stage, lane, done, acc); });
    }
  } else if (g.w != nullptr) {
    Main rows;
    rows.lds = lds + wave * Main::kBytes;
    rows.bytes = g.in_dim * sizeof(E);
    rows.piece = piece;
    rows.base_a = reinterpret_cast<const unsigned char*>(static_cast<const E*>(g.w) + static_cast<uint64_t>(n0) * g.in_dim);
    rows.base_b = x;
    rows.off_b[0] = x_row;
#pragma unroll
    for (int i = 0; i < 2; ++i) rows.off_a[i] = min(8 * i + lane / 8, g.out_dim - 1 - n0) * rows.bytes + piece;
    rows.Run(kStepBytes * wave, kStepBytes * kWaves, [&](const unsigned char* stage, auto&& done) {
      u32x4_t w[2], v[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        w[p] = StagePiece(stage, lane % 16, 4 * p + lane / 16);
        v[p] = StagePiece(stage, 16 + lane % kFewRows, 4 * p + lane / 16);
      }
      done();
#pragma unroll
      for (int p = 0; p < 2; ++p) acc[0][0] = Mma16<E>(w[p], v[p], acc[0][0]);
    });
  }
  auto* part = reinterpret_cast<f32x4_t(*)[64]>(lds);
  __syncthreads();
  part[wave][lane] = acc[0][0];
  __syncthreads();
  if (wave != kWaves + kSide - 1) return;

  // Lane l: row t = l % 16, outputs (of the product) or ranks (of the low-rank rows) 4 (l / 16) .. + 3.
  const uint32_t first = 4 * (lane / 16);
  f32x4_t low = part[kWaves][lane];
#pragma unroll
  for (int i = 1; i < kSide; ++i) low += part[kWaves + i][lane];
  if constexpr (kIsE4m3<E>) scale *= x_scale;
  const uint32_t of = first / g.max_rank;  // the sequence of these four ranks
  const uint32_t its_rank = its == 0 ? rank[0] : its == 1 ? rank[1] : 0;
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) {
    const bool kept = static_cast<int32_t>(of) == its && first + e - of * g.max_rank < its_rank;
    u[t][first + e] = kept ? low[e] * scale : 0.0f;
  }
  WaveSync();
  const uint32_t j = kPer * (lane / 16);
  f32x4_t ur[kPer / 4] = {};
  if (j < kFewRanks) {
#pragma unroll
    for (uint32_t i = 0; i < kPer / 4; ++i) ur[i] = *reinterpret_cast<const f32x4_t*>(&u[t][j + 4 * i]);
  }
  f32x4_t v = {0, 0, 0, 0};
  const uint32_t parts = sizeof(Low) == 2 ? g.parts : 1;
#pragma unroll 1
  for (uint32_t p = 0; p < parts; ++p) {
    const u32x4_t pu = NextPart<Low>(ur);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      const auto left = static_cast<int32_t>(rank[i] + i * g.max_rank) - static_cast<int32_t>(j);
      const f32x4_t d = Mma16<Low>(First<Low>(b[i], left), pu, f32x4_t{0, 0, 0, 0});
      if (its == static_cast<int32_t>(i)) v += d;
    }
  }
  const uint32_t n = n0 + first;
  if (its == kNoRow || n >= g.out_dim) return;
  f32x4_t sum = part[0][lane];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) sum += part[w][lane];
  if constexpr (kIsE4m3<E>) {
    if (g.w != nullptr) sum = Rescaled(g, x_scale, n, sum);
  }
  Store(g, t, n, sum + v);
}

// ---- The product by tiles ------------------------------------------------------------------------------------------------
//
// One workgroup: 32 kN kWN outputs x 32 kT kWT rows, its wavefronts in a kWN x kWT grid of 32 kN x 32 kT each, kept in
// accumulators. 128 bytes of the inner dimension at a time are copied from memory straight into LDS (global_load_lds, no
// registers), kStages steps ahead. A row's eight 16-byte pieces lie in LDS at piece p ^ (row / 2 % 8): 32 rows of 128 bytes
// read at one piece are then free of bank conflicts (with p ^ (row % 8) each read takes half as long again). The copy
// writes LDS in lane order, so it is the lanes' source addresses that are permuted.
//
// Bound by the matrix instructions and what keeps them fed. 15,000 rows, 4096 to 4096 channels, bf16, rank 64: about 435 us of
// 256 x 256 tiles, 1.16 PFLOP/s, where a plain library product of these sizes takes 356 us; 944 tiles are 3.7 rounds of the
// CUs, the instructions and their LDS reads by themselves 365 us, the copies 60 and the last store 50 more. e4m3 rows, 6,700 x
// 4096 x 12288, rank 32: 2.0 PFLOP/s.

// Every copy but this wavefront's last kLeft has landed, its own LDS reads have returned, and then every wavefront's.
template <int kLeft>
__device__ __forceinline__ void WaitStep() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLeft) : "memory");
}

// Adapters that a tile of 64 x 64 takes step by step; more are added element by element, whose time grows with the rank where
// a step's does not. 100 rows, 4096 to 12288: 16 adapters of rank 16 59 us by steps and 53 by elements, 64 of them 79 and 57;
// 16 of rank 64 71 and 90, 64 of them 104 and 107.
__device__ __forceinline__ uint32_t AdaptersBySteps(uint32_t max_rank) { return max(4u, max_rank / 4); }

template <typename E, int kN, int kT, int kWN, int kWT, int kStages>
__global__ void __launch_bounds__(64 * kWN * kWT, 1)
TileKernel(LoraArgs g, uint32_t n_tiles, uint32_t t_tiles, uint32_t first) {
  constexpr int kWaves = kWN * kWT;
  constexpr int kRowsN = 32 * kN * kWN, kRowsT = 32 * kT * kWT;
  constexpr int kCopiesN = kRowsN / (8 * kWaves), kCopiesT = kRowsT / (8 * kWaves);  // of 8 rows, by each wavefront
  constexpr uint32_t kStage = (kRowsN + kRowsT) * kStepBytes;
  static_assert(kWaves % 2 == 0 && kRowsN % 16 == 0, "the permutation of a wavefront's copies is the same for each");
  static_assert(kCopiesN * 8 * kWaves == kRowsN && kCopiesT * 8 * kWaves == kRowsT, "every wavefront copies whole rows");
  __shared__ __align__(16) unsigned char lds[kStages * kStage];
  __shared__ int32_t slot[kRowsT];
  __shared__ int32_t adapter[kRowsT];  // of the tile's rows, each once
  __shared__ uint32_t adapter_rank[kRowsT], adapter_count;
  __shared__ __align__(16) float w_scale[kIsE4m3<E> ? kRowsN : 4];
  const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);

  // Workgroups go to the 8 XCDs in turn; each XCD takes one run of the tiles, ordered in blocks of kBlockT rows of tiles,
  // so that the tiles in flight on an XCD share weight and token rows in its L2.
  constexpr uint32_t kXcds = 8, kBlockT = 8;
  const uint32_t tiles = n_tiles * t_tiles;
  const uint32_t per_xcd = (tiles + kXcds - 1) / kXcds;
  const uint32_t at = (blockIdx.x % kXcds) * per_xcd + blockIdx.x / kXcds;
  if (blockIdx.x / kXcds >= per_xcd || at >= tiles) return;
  const uint32_t block = at / (kBlockT * n_tiles);
  const uint32_t block_rows = min(kBlockT, t_tiles - block * kBlockT);
  const uint32_t in_block = at - block * kBlockT * n_tiles;
  const uint32_t t0 = first + (block * kBlockT + in_block % block_rows) * kRowsT;
  const uint32_t n0 = (in_block / block_rows) * kRowsN;

  f32x16_t acc[kN][kT];
#pragma unroll
  for (int n = 0; n < kN; ++n) {
#pragma unroll
    for (int t = 0; t < kT; ++t) acc[n][t] = f32x16_t{};
  }
  const uint32_t wn = (wave % kWN) * 32 * kN, wt = (wave / kWN) * 32 * kT;  // this wavefront's corner of the tile

  // The copies. Rows past the last output or token repeat the last one; what they give is not stored.
  using Low = LowOf<E>;
  const uint32_t bytes = g.in_dim * sizeof(E);
  const uint64_t x_bytes = g.x_stride * sizeof(E);
  const uint32_t full = g.w != nullptr ? bytes / kStepBytes : 0;
  const uint32_t steps = g.w != nullptr ? (bytes + kStepBytes - 1) / kStepBytes : 0;
  const auto* w_base = static_cast<const unsigned char*>(g.w) + static_cast<uint64_t>(n0) * bytes;
  const auto* x_base = static_cast<const unsigned char*>(g.x) + t0 * x_bytes;
  const uint32_t last_n = g.out_dim - 1 - n0, last_t = g.tokens - 1 - t0;
  const uint32_t piece = 16 * ((lane % 8) ^ (4 * (wave % 2) + lane / 16));  // rows 8 (wave + kWaves i) + lane / 8
  uint32_t off_n[kCopiesN], off_t[kCopiesT];
#pragma unroll
  for (int i = 0; i < kCopiesN; ++i) off_n[i] = min(8 * (wave + kWaves * i) + lane / 8, last_n) * bytes + piece;
#pragma unroll
  for (int i = 0; i < kCopiesT; ++i) {
    off_t[i] = min(8 * (wave + kWaves * i) + lane / 8, last_t) * static_cast<uint32_t>(x_bytes) + piece;
  }
  const uint32_t lds0 = LdsAddress(lds);
  const auto zero = [&](uint32_t stage) {  // this lane's pieces of a stage
#pragma unroll
    for (int i = 0; i < kCopiesN + kCopiesT; ++i) {
      *reinterpret_cast<u32x4_t*>(lds + stage * kStage + 1024 * (wave + kWaves * i) + 16 * lane) = u32x4_t{0, 0, 0, 0};
    }
  };
  const auto copy = [&](uint32_t step) {
    const uint32_t to_n = lds0 + (step % kStages) * kStage + 1024 * wave, to_t = to_n + kRowsN * kStepBytes;
    const uint32_t from = step * kStepBytes;
    if (step < full) {
#pragma unroll
      for (int i = 0; i < kCopiesN; ++i) Copy16(w_base + from, off_n[i], to_n + 1024 * kWaves * i);
#pragma unroll
      for (int i = 0; i < kCopiesT; ++i) Copy16(x_base + from, off_t[i], to_t + 1024 * kWaves * i);
    } else if (from + piece < bytes) {
#pragma unroll
      for (int i = 0; i < kCopiesN; ++i) Copy16(w_base + from, off_n[i], to_n + 1024 * kWaves * i);
#pragma unroll
      for (int i = 0; i < kCopiesT; ++i) Copy16(x_base + from, off_t[i], to_t + 1024 * kWaves * i);
    } else {  // the last, partial step: pieces past the row's end are zeros
      zero(step % kStages);
    }
  };
#pragma unroll
  for (uint32_t i = 0; i < kStages; ++i) {
    if (i < steps) copy(i);
  }
  FillSlots(g, t0, kRowsT, slot);
  if constexpr (kIsE4m3<E>) {
    if (g.w != nullptr) {
      for (uint32_t i = threadIdx.x; i < kRowsN; i += 64 * kWaves) w_scale[i] = g.w_scale[min(n0 + i, g.out_dim - 1)];
    }
  }
  __syncthreads();
  if (wave == 0 && g.a != nullptr) {
    int32_t its[kRowsT / 64];
    uint32_t count = 0;
#pragma unroll
    for (int c = 0; c < kRowsT / 64; ++c) its[c] = slot[64 * c + lane];
#pragma unroll
    for (int c = 0; c < kRowsT / 64; ++c) {
      for (uint64_t left = __ballot(its[c] >= 0); left != 0; left = __ballot(its[c] >= 0)) {
        const int32_t one = __builtin_amdgcn_readlane(its[c], __builtin_ctzll(left));
        if (lane == 0) adapter[count] = one;
        ++count;
#pragma unroll
        for (int k = c; k < kRowsT / 64; ++k) its[k] = its[k] == one ? kNoAdapter : its[k];
      }
    }
    WaveSync();
    for (uint32_t i = lane; i < count; i += 64) adapter_rank[i] = RankOf(g, adapter[i]);
    if (lane == 0) adapter_count = count;
  }

  // A step is consumed in kPhases phases of kPieces pieces a lane, each in kHalves parts of the wavefront's rows; the
  // operands are read from LDS one part ahead of the products that use them. The last part waits for the next step's
  // copies, reads its first operands and refills the buffer that every wavefront has then read, all under its own products.
  uint32_t at_piece[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) at_piece[p] = (lane % 32) * kStepBytes + 16 * ((2 * p + lane / 32) ^ (lane / 2 % 8));
  constexpr int kCopies = kCopiesN + kCopiesT;
  if (steps > 0) {
    constexpr int kPieces = std::is_same_v<E, E4m3> ? 2 : 1, kPhases = 4 / kPieces;
    // e4m3 operands take twice the registers, so half of the rows at a time.
    constexpr int kHalves = kPieces == 2 && kT > 1 ? 2 : 1, kHalfT = kT / kHalves, kParts = kPhases * kHalves;
    FragOf<E> fn[2][kN], ft[2][kHalfT];
    const auto load = [&](const unsigned char* rows, int phase) -> FragOf<E> {
      if constexpr (kPieces == 2) {
        const u32x4_t lo = *reinterpret_cast<const u32x4_t*>(rows + at_piece[2 * phase]);
        const u32x4_t hi = *reinterpret_cast<const u32x4_t*>(rows + at_piece[2 * phase + 1]);
        return __builtin_bit_cast(i32x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      } else {
        return *reinterpret_cast<const u32x4_t*>(rows + at_piece[phase]);
      }
    };
    const auto read = [&](const unsigned char* from, int part) {
      const int phase = part / kHalves, half = part % kHalves;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        if (half == 0) fn[phase % 2][n] = load(from + (wn + 32 * n) * kStepBytes, phase);
      }
#pragma unroll
      for (int t = 0; t < kHalfT; ++t) {
        ft[part % 2][t] = load(from + (kRowsN + wt + 32 * (half * kHalfT + t)) * kStepBytes, phase);
      }
    };
    if (steps >= kStages) {
      WaitStep<(kStages - 1) * kCopies>();
    } else {
      WaitStep<0>();
    }
    read(lds, 0);
#pragma unroll 1
    for (uint32_t step = 0; step < steps; ++step) {
      const unsigned char* from = lds + (step % kStages) * kStage;
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        if (part + 1 < kParts) {
          read(from, part + 1);
        } else if (step + 1 < steps) {
          // Of the kStages steps whose copies are out, the next one's are to have landed.
          if (kStages > 2 && step + kStages - 1 < steps) {
            WaitStep<(kStages - 2) * kCopies>();
          } else {
            WaitStep<0>();
          }
          read(lds + ((step + 1) % kStages) * kStage, 0);
          if (step + kStages >= full && step + kStages < steps) copy(step + kStages);
        }
        // The next stage's copies go out one after each of the last part's products.
        const bool refill = part + 1 == kParts && step + kStages < full;
        const uint32_t to = lds0 + (step % kStages) * kStage + 1024 * wave, ahead = (step + kStages) * kStepBytes;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < kN; ++n) {
#pragma unroll
          for (int t = 0; t < kHalfT; ++t) {
            f32x16_t& sum = acc[n][(part % kHalves) * kHalfT + t];
            sum = Mma32<E>(fn[part / kHalves % 2][n], ft[part % 2][t], sum);
            // Keeps the products of a part between its reads and the next part's.
            if constexpr (kN * kT >= 8) asm volatile("" : "+v"(sum));
            constexpr int kEach = (kCopies + kN * kHalfT - 1) / (kN * kHalfT);  // copies after each product
#pragma unroll
            for (int c = (n * kHalfT + t) * kEach; c < (n * kHalfT + t + 1) * kEach && c < kCopies; ++c) {
              if (!refill) continue;
              if (c < kCopiesN) {
                Copy16(w_base + ahead, off_n[c < kCopiesN ? c : 0], to + 1024 * kWaves * c);
              } else {
                Copy16(x_base + ahead, off_t[c < kCopiesN ? 0 : c - kCopiesN], to + 1024 * kWaves * c);
              }
            }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  __syncthreads();  // the stages are free, the adapters known

  // The adapters of the tile, one after the other, by the same steps: 128 bytes of the ranks of the adapter's outputs and of
  // the low-rank rows. A row takes only its own adapter's sums, so that no adapter's values, whatever they are, reach
  // another's rows. acc[n][t], register i, lane l: row wt + 32 t + l % 32, output wn + 32 n + 8 (i / 4) + 4 (l / 32) + i % 4.
  if constexpr (kIsE4m3<E>) {
    if (g.w != nullptr) {
#pragma unroll
      for (int t = 0; t < kT; ++t) {
        const float xs = g.x_scale[t0 + min(wt + 32 * t + lane % 32, last_t)];
#pragma unroll
        for (int n = 0; n < kN; ++n) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x4_t ws = *reinterpret_cast<const f32x4_t*>(w_scale + wn + 32 * n + 8 * q + 4 * (lane / 32));
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][t][4 * q + e] *= xs * ws[e];
          }
        }
      }
    }
  }
  // Below, a lane stores 8 outputs of a row; the addends of whole eights are loaded ahead: before the adapters where there
  // are registers for it, else after them.
  constexpr uint32_t kOctets = 4 * kN, kRowsAtOnce = 64 / kOctets, kTurns = 32 / kRowsAtOnce;
  constexpr bool kEarly = kN * kT <= 4;
  const uint32_t out = n0 + wn + 8 * (lane % kOctets);
  const bool whole = out + 8 <= g.out_dim, part = out < g.out_dim && !whole;
  u32x4_t early[kT][kTurns];
  const auto load_addends = [&] {
#pragma unroll
    for (int t = 0; t < kT; ++t) {
#pragma unroll
      for (uint32_t k = 0; k < kTurns; ++k) {
        const uint32_t row = wt + 32 * t + kRowsAtOnce * k + lane / kOctets;
        early[t][k] = u32x4_t{0, 0, 0, 0};
        if (g.addend != nullptr && !g.addend_f32 && whole && slot[row] != kNoRow) {
          const uint64_t at = (t0 + row) * g.addend_stride + out;
          early[t][k] = *reinterpret_cast<const Bf16x8*>(static_cast<const uint16_t*>(g.addend) + at);
        }
      }
    }
  };
  if (kEarly) load_addends();
  const uint32_t count = __builtin_amdgcn_readfirstlane(g.a != nullptr ? adapter_count : 0);
  if (kN * kT > 1 || count <= AdaptersBySteps(g.max_rank)) {
    constexpr int kPer = 16 / sizeof(Low);
    const uint32_t row_bytes = g.max_rank * sizeof(Low);
    const uint32_t parts = sizeof(Low) == 2 ? g.parts : 1;
    // A place in the list of steps: adapter, part of the low-rank rows, first byte of their ranks.
    struct Place {
      uint32_t index, part, from;
      int32_t slot;
      uint32_t bytes;  // of the adapter's ranks
    };
    const auto enter = [&](Place& p) {  // the next adapter with a rank, from p.index on
      for (; p.index < count; ++p.index) {
        p.slot = __builtin_amdgcn_readfirstlane(adapter[p.index]);
        p.bytes = __builtin_amdgcn_readfirstlane(adapter_rank[p.index]) * sizeof(Low);
        if (p.bytes > 0) break;
      }
      p.part = p.from = 0;
    };
    const auto advance = [&](Place& p) {
      p.from += kStepBytes;
      if (p.from < p.bytes) return;
      p.from = 0;
      if (++p.part < parts) return;
      ++p.index;
      enter(p);
    };
    const auto copy_low = [&](const Place& p, uint32_t stage) {
      const uint32_t to_n = lds0 + stage * kStage + 1024 * wave, to_t = to_n + kRowsN * kStepBytes;
      const uint32_t at = p.from + piece;
      if (at >= p.bytes) return;  // what the stage holds there is not multiplied
      // A row of the pool is at most 512 bytes, so a tile's are within 32 bits of its first.
      const uint64_t b_row = static_cast<uint64_t>(p.slot) * g.out_dim + n0;
      const auto* b_base = static_cast<const unsigned char*>(g.b) + b_row * row_bytes;
      const auto* u_base = sizeof(Low) == 2 ? reinterpret_cast<const unsigned char*>(g.u_bf16 + p.part * g.u_part)
                                            : reinterpret_cast<const unsigned char*>(g.u);
      u_base += t0 * static_cast<uint64_t>(row_bytes);
#pragma unroll
      for (int i = 0; i < kCopiesN; ++i) {
        Copy16(b_base, min(8 * (wave + kWaves * i) + lane / 8, last_n) * row_bytes + at, to_n + 1024 * kWaves * i);
      }
#pragma unroll
      for (int i = 0; i < kCopiesT; ++i) {
        Copy16(u_base, min(8 * (wave + kWaves * i) + lane / 8, last_t) * row_bytes + at, to_t + 1024 * kWaves * i);
      }
    };
    int32_t row_slot[kT];
#pragma unroll
    for (int t = 0; t < kT; ++t) row_slot[t] = slot[wt + 32 * t + lane % 32];
    Place next{}, now{};
    enter(next);
    now = next;
    uint32_t step = 0;
#pragma unroll 1
    for (uint32_t i = 0; i + 1 < kStages && next.index < count; ++i, advance(next)) copy_low(next, i);
#pragma unroll 1
    for (; now.index < count; advance(now), ++step) {
      if constexpr (kStages == 1) {
        __syncthreads();  // the step before is read
        copy_low(now, 0);
        WaitStep<0>();
      } else {
        WaitStep<0>();
        if (next.index < count) {
          copy_low(next, (step + kStages - 1) % kStages);
          advance(next);
        }
      }
      const unsigned char* from = lds + (step % kStages) * kStage;
#pragma unroll
      for (int t = 0; t < kT; ++t) {
        const bool mine = row_slot[t] == now.slot;
        if (__ballot(mine) == 0) continue;
        f32x16_t d[kN];
#pragma unroll
        for (int n = 0; n < kN; ++n) d[n] = f32x16_t{};
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          if (now.from + 32 * p >= now.bytes) break;
          const auto left = static_cast<int32_t>(now.bytes / sizeof(Low)) -
                            static_cast<int32_t>(now.from / sizeof(Low) + kPer * (2 * p + lane / 32));
          const u32x4_t fu =
              First<Low>(*reinterpret_cast<const u32x4_t*>(from + at_piece[p] + (kRowsN + wt + 32 * t) * kStepBytes), left);
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            const u32x4_t fb =
                First<Low>(*reinterpret_cast<const u32x4_t*>(from + at_piece[p] + (wn + 32 * n) * kStepBytes), left);
            d[n] = Mma32<Low>(fb, fu, d[n]);
          }
        }
#pragma unroll
        for (int n = 0; n < kN; ++n) {
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[n][t][i] += mine ? d[n][i] : 0.0f;
        }
      }
    }
    __syncthreads();
  } else if constexpr (kN * kT == 1) {
    const uint32_t token = t0 + min(wt + lane % 32, last_t);
    const int32_t s = slot[wt + lane % 32];
    const uint32_t rank = RankOf(g, s);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f32x4_t v = {acc[0][0][4 * q], acc[0][0][4 * q + 1], acc[0][0][4 * q + 2], acc[0][0][4 * q + 3]};
      AddLowRank<Low>(g, token, n0 + wn + 8 * q + 4 * (lane / 32), max(s, 0), rank, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[0][0][4 * q + e] = v[e];
    }
  }

  // The sums go through LDS by 32 rows, each wavefront in a part of its own, and from there whole 128-byte runs of a row to
  // a store. bf16 addends of all the rows are requested before the first is used (f32 ones of 32 rows, to save registers).
  constexpr uint32_t kRowWords = 32 * kN + 4;  // 4 words of padding put 8 neighbouring rows on different banks
  static_assert(kWaves * 32 * kRowWords * 4 <= kStages * kStage, "the wavefronts' parts fit the stages");
  float* mine = reinterpret_cast<float*>(lds) + wave * 32 * kRowWords;
  if (!kEarly) load_addends();
#pragma unroll
  for (int t = 0; t < kT; ++t) {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        *reinterpret_cast<f32x4_t*>(mine + (lane % 32) * kRowWords + 32 * n + 8 * q + 4 * (lane / 32)) =
            f32x4_t{acc[n][t][4 * q], acc[n][t][4 * q + 1], acc[n][t][4 * q + 2], acc[n][t][4 * q + 3]};
      }
    }
    WaveSync();
#pragma unroll
    for (uint32_t k = 0; k < kTurns; ++k) {
      const uint32_t row = kRowsAtOnce * k + lane / kOctets;
      const float* from = mine + row * kRowWords + 8 * (lane % kOctets);
      const bool live = slot[wt + 32 * t + row] != kNoRow;
      const uint64_t token = t0 + wt + 32 * t + row;
      if (whole && live) {
        f32x4_t lo = *reinterpret_cast<const f32x4_t*>(from), hi = *reinterpret_cast<const f32x4_t*>(from + 4);
        if (g.addend_f32) {
          const auto* p = reinterpret_cast<const F32x4*>(static_cast<const float*>(g.addend) + token * g.addend_stride + out);
          lo += p[0];
          hi += p[1];
        } else {
          const u32x4_t w = early[t][k];
          lo += f32x4_t{Bf16LoToF32(w[0]), Bf16HiToF32(w[0]), Bf16LoToF32(w[1]), Bf16HiToF32(w[1])};
          hi += f32x4_t{Bf16LoToF32(w[2]), Bf16HiToF32(w[2]), Bf16LoToF32(w[3]), Bf16HiToF32(w[3])};
        }
        if (g.y_f32) {
          auto* p = reinterpret_cast<F32x4*>(static_cast<float*>(g.y) + token * g.y_stride + out);
          p[0] = lo;
          p[1] = hi;
        } else {
          *reinterpret_cast<Bf16x8*>(static_cast<uint16_t*>(g.y) + token * g.y_stride + out) =
              Bf16x8{PackBf16Rne(lo[0], lo[1]), PackBf16Rne(lo[2], lo[3]), PackBf16Rne(hi[0], hi[1]),
                     PackBf16Rne(hi[2], hi[3])};
        }
      }
    }
    if (part) {  // the last outputs of rows that do not end with a whole eight
#pragma unroll 1
      for (uint32_t row = lane / kOctets; row < 32; row += kRowsAtOnce) {
        const uint64_t token = t0 + wt + 32 * t + row;
        if (slot[wt + 32 * t + row] == kNoRow) continue;
#pragma unroll 1
        for (uint32_t e = 0; e < g.out_dim - out; ++e) {
          const float add = g.addend != nullptr ? AddendOne(g, token * g.addend_stride + out + e) : 0.0f;
          StoreOne(g, token * g.y_stride + out + e, mine[row * kRowWords + 8 * (lane % kOctets) + e] + add);
        }
      }
    }
    WaveSync();
  }
}

// ---- Admission -----------------------------------------------------------------------------------------------------------

bool FloatType(uint32_t dt) { return dt == ROOST_DTYPE_BF16 || dt == ROOST_DTYPE_F32; }
uint64_t Stride(uint32_t stride, uint32_t dim) { return stride == 0 ? dim : stride; }

struct Extent {
  uintptr_t first, end;
};
Extent ExtentOf(const RoostDeviceSpan& s, uint64_t elems) {
  const auto a = reinterpret_cast<uintptr_t>(s.address);
  return Extent{a, a == 0 ? a : a + elems * roost::ElementBytes(s.dtype)};
}
bool Overlap(Extent a, Extent b) { return a.first < b.end && b.first < a.end; }

// Elements that [rows, dim] at `stride` elements a row reaches.
uint64_t Reach(uint64_t rows, uint64_t dim, uint64_t stride) { return rows == 0 ? 0 : (rows - 1) * stride + dim; }

// The shape's rules; the spans' addresses are looked at only by run().
RoostStatus Admit(const RoostAmdGemmLoraParams& p, bool for_run) {
  roost::Gate gate(kOp);
  const uint32_t e = p.x.dtype;
  const bool eight = e == ROOST_DTYPE_F8E4M3, shared = p.weight.address != nullptr, lora = p.lora_a.address != nullptr;
  const uint32_t low = e == ROOST_DTYPE_F32 ? ROOST_DTYPE_F32 : ROOST_DTYPE_BF16;
  gate.Expect(p.reserved0 == 0, ROOST_STATUS_INVALID_ARGUMENT, "reserved0 = %u, must be 0", p.reserved0)
      .Expect(FloatType(e) || eight, ROOST_STATUS_UNSUPPORTED, "x is %s; built for bf16, f32 and f8e4m3 rows",
              roost::Describe(e).name)
      .Expect(shared || lora, ROOST_STATUS_INVALID_ARGUMENT, "neither a weight nor adapters were given")
      .Expect(p.in_dim > 0 && p.out_dim > 0 && p.in_dim <= 1u << 20 && p.out_dim <= 1u << 20, ROOST_STATUS_UNSUPPORTED,
              "in_dim = %u, out_dim = %u; built for 1 to 1,048,576", p.in_dim, p.out_dim)
      .Expect(p.tokens < 1u << 20 && p.batch <= p.tokens + 65536u, ROOST_STATUS_UNSUPPORTED,
              "tokens = %u, batch = %u; built for up to 1,048,575 rows", p.tokens, p.batch)
      .Expect(lora || (p.adapters == 0 && p.max_rank == 0), ROOST_STATUS_INVALID_ARGUMENT,
              "adapters = %u, max_rank = %u without lora_a", p.adapters, p.max_rank)
      .Expect(!lora || (p.adapters > 0 && p.max_rank > 0 && p.max_rank % 8 == 0 && p.max_rank <= kMaxRank),
              ROOST_STATUS_UNSUPPORTED, "adapters = %u, max_rank = %u; built for ranks that are multiples of 8 up to %u",
              p.adapters, p.max_rank, kMaxRank);
  ROOST_GATE_RETURN(gate);
  const uint64_t es = roost::ElementBytes(e);
  const uint64_t x_stride = Stride(p.x_stride, p.in_dim), y_stride = Stride(p.output_stride, p.out_dim);
  const uint64_t add_stride = Stride(p.addend_stride, p.out_dim);
  gate.Expect(p.in_dim * es % 16 == 0 && x_stride * es % 16 == 0, ROOST_STATUS_UNSUPPORTED,
              "in_dim = %u, x_stride = %llu: rows of %s must be multiples of 16 bytes", p.in_dim,
              static_cast<unsigned long long>(x_stride), roost::Describe(e).name)
      .Expect(x_stride <= 1u << 20, ROOST_STATUS_UNSUPPORTED, "x_stride = %llu; built for up to 1,048,576",
              static_cast<unsigned long long>(x_stride))
      .Expect(x_stride >= p.in_dim && y_stride >= p.out_dim && add_stride >= p.out_dim, ROOST_STATUS_INVALID_ARGUMENT,
              "a row stride (x %llu, output %llu, addend %llu) is below its row's width",
              static_cast<unsigned long long>(x_stride), static_cast<unsigned long long>(y_stride),
              static_cast<unsigned long long>(add_stride));
  if (!gate.ok() || !for_run) return gate.status();
  const uint64_t x_elems = Reach(p.tokens, p.in_dim, x_stride), y_elems = Reach(p.tokens, p.out_dim, y_stride);
  const uint64_t add_elems = Reach(p.tokens, p.out_dim, add_stride);
  const uint64_t w_elems = static_cast<uint64_t>(p.out_dim) * p.in_dim;
  const uint64_t pool = static_cast<uint64_t>(p.adapters) * p.max_rank;
  gate.Expect(e == ROOST_DTYPE_F32 ? p.output.dtype == e : FloatType(p.output.dtype), ROOST_STATUS_UNSUPPORTED,
              "output is %s beside %s rows", roost::Describe(p.output.dtype).name, roost::Describe(e).name)
      .Tensor("x", p.x, e, x_elems)
      .Tensor("output", p.output, p.output.dtype, y_elems)
      .Tensor("cu_seqlens", p.cu_seqlens, ROOST_DTYPE_I32, p.batch + 1ull)
      .Aligned("x", p.x.address, 16)
      .Aligned("output", p.output.address, roost::ElementBytes(p.output.dtype))
      .Aligned("cu_seqlens", p.cu_seqlens.address, 4);
  ROOST_GATE_RETURN(gate);
  if (eight) {
    gate.Tensor("x_scale", p.x_scale, ROOST_DTYPE_F32, p.tokens).Aligned("x_scale", p.x_scale.address, 4);
    if (shared) gate.Tensor("w_scale", p.w_scale, ROOST_DTYPE_F32, p.out_dim).Aligned("w_scale", p.w_scale.address, 4);
  } else {
    gate.Expect(p.x_scale.address == nullptr && p.w_scale.address == nullptr, ROOST_STATUS_INVALID_ARGUMENT,
                "x_scale and w_scale belong to f8e4m3 rows; x is %s", roost::Describe(e).name);
  }
  if (gate.ok() && shared) gate.Tensor("weight", p.weight, e, w_elems).Aligned("weight", p.weight.address, 16);
  if (gate.ok() && lora) {
    gate.Tensor("lora_a", p.lora_a, low, pool * p.in_dim)
        .Tensor("lora_b", p.lora_b, low, pool * p.out_dim)
        .Tensor("lora_slots", p.lora_slots, ROOST_DTYPE_I32, p.batch)
        .OptionalTensor("lora_scale", p.lora_scale, ROOST_DTYPE_F32, p.adapters)
        .OptionalTensor("ranks", p.ranks, ROOST_DTYPE_I32, p.adapters)
        .Aligned("lora_a", p.lora_a.address, 16)
        .Aligned("lora_b", p.lora_b.address, 16)
        .Aligned("lora_slots", p.lora_slots.address, 4)
        .Aligned("lora_scale", p.lora_scale.address, 4)
        .Aligned("ranks", p.ranks.address, 4);
  }
  const bool adds = p.addend.address != nullptr;
  if (gate.ok() && adds) {
    gate.Expect(FloatType(p.addend.dtype), ROOST_STATUS_UNSUPPORTED, "addend is %s; built for bf16 and f32",
                roost::Describe(p.addend.dtype).name);
    if (gate.ok()) {
      gate.Tensor("addend", p.addend, p.addend.dtype, add_elems)
          .Aligned("addend", p.addend.address, roost::ElementBytes(p.addend.dtype));
    }
  }
  ROOST_GATE_RETURN(gate);
  const Extent y = ExtentOf(p.output, y_elems);
  const bool in_place = adds && p.addend.address == p.output.address && p.addend.dtype == p.output.dtype &&
                        add_stride == y_stride;
  gate.Expect(!adds || in_place || !Overlap(y, ExtentOf(p.addend, add_elems)), ROOST_STATUS_INVALID_ARGUMENT,
              "output overlaps the addend without being exactly that span");
  const Extent read[] = {ExtentOf(p.x, x_elems),           ExtentOf(p.weight, w_elems),
                         ExtentOf(p.lora_a, pool * p.in_dim), ExtentOf(p.lora_b, pool * p.out_dim),
                         ExtentOf(p.x_scale, p.tokens),    ExtentOf(p.w_scale, p.out_dim),
                         ExtentOf(p.lora_scale, p.adapters), ExtentOf(p.ranks, p.adapters),
                         ExtentOf(p.lora_slots, p.batch),  ExtentOf(p.cu_seqlens, p.batch + 1ull)};
  for (const Extent& r : read) {
    gate.Expect(!Overlap(y, r), ROOST_STATUS_INVALID_ARGUMENT, "output overlaps an input of the call");
  }
  return gate.status();
}

// The low-rank rows in f32, then, beside bf16 adapters, in bf16: one rounding under a bf16 output, three parts, which hold
// all 24 bits, under an f32 one.
uint64_t LowRankElements(const RoostAmdGemmLoraParams& p) {
  return p.lora_a.address == nullptr ? 0 : roost::RoundUp(static_cast<uint64_t>(p.tokens) * p.max_rank, 64);
}
uint32_t LowRankParts(const RoostAmdGemmLoraParams& p) {
  return p.x.dtype == ROOST_DTYPE_F32 ? 0 : p.output.dtype == ROOST_DTYPE_F32 ? 3 : 1;
}
uint64_t WorkspaceBytes(const RoostAmdGemmLoraParams& p) {
  return LowRankElements(p) * (sizeof(float) + LowRankParts(p) * sizeof(uint16_t));
}

// ---- Launch --------------------------------------------------------------------------------------------------------------

template <typename E, int kT, int kR>
void LaunchShrink(const LoraArgs& g, hipStream_t stream) {
  // One tile: two workgroups share a CU's LDS. Else eight wavefronts where three stages of theirs fit, then as many stages
  // as there is room for, up to four.
  constexpr bool kOne = kT == 1 && kR == 1;
  constexpr int kStepRows = 16 * kT + 16 * kR * static_cast<int>(sizeof(LowOf<E>) / sizeof(E));
  constexpr int kRoom = (kOne ? 75 : 150) * 1024;
  constexpr int kWaves = 8 * (kOne ? 2 : 3) * kStepRows * static_cast<int>(kStepBytes) <= kRoom ? 8 : 4;
  constexpr int kStages = std::min(4, kRoom / (kWaves * kStepRows * static_cast<int>(kStepBytes)));
  static_assert(kStages >= 2, "a step on its way while one is multiplied");
  const dim3 grid(roost::CeilDiv(g.tokens, 16 * kT) + g.batch, roost::CeilDiv(g.max_rank, 16 * kR));
  hipLaunchKernelGGL((ShrinkKernel<E, kT, kR, kWaves, kStages>), grid, dim3(64 * kWaves), 0, stream, g);
}
template <typename E, int kT>
void LaunchShrinkOfRows(const LoraArgs& g, hipStream_t stream) {
  // Blocks of 16 ranks while all the workgroups have a CU of their own, else as wide as the pool's ranks, up to 32 or 64,
  // so that the rows are read once. 64 one-token sequences of 4096 channels, rank 32: 17.8 us a call in blocks of 16, 18.7
  // of 32; 256 of them 24.9 and 22.5; 1,000 of rank 128: 186 in blocks of 16, 127 of 64.
  const uint64_t blocks = (roost::CeilDiv(g.tokens, 16 * kT) + g.batch) * roost::CeilDiv(g.max_rank, 16);
  if (g.max_rank <= 16 || (kT == 1 && blocks <= kCus)) return LaunchShrink<E, kT, 1>(g, stream);
  if constexpr (!kIsE4m3<E>) {
    if (g.max_rank > 32) return LaunchShrink<E, kT, 4>(g, stream);
  }
  return LaunchShrink<E, kT, 2>(g, stream);
}

template <typename E, int kN, int kT, int kWaves, int kLow, int kStages>
void LaunchProduct(const LoraArgs& g, hipStream_t stream) {
  const auto n_tiles = static_cast<uint32_t>(roost::CeilDiv(g.out_dim, 16 * kN));
  const auto grid = static_cast<uint32_t>(n_tiles * roost::CeilDiv(g.tokens, 16 * kT));
  hipLaunchKernelGGL((ProductKernel<E, kN, kT, kWaves, kLow, kStages>), dim3(grid), dim3(64 * (kWaves + kLow)), 0, stream, g,
                     n_tiles);
}

// Rows first .. end - 1.
template <typename E, int kN, int kT, int kWN, int kWT, int kStages>
void LaunchTiles(const LoraArgs& g, uint32_t first, uint32_t end, hipStream_t stream) {
  const auto n_tiles = static_cast<uint32_t>(roost::CeilDiv(g.out_dim, 32 * kN * kWN));
  const auto t_tiles = static_cast<uint32_t>(roost::CeilDiv(end - first, 32 * kT * kWT));
  const auto grid = static_cast<uint32_t>(roost::RoundUp(n_tiles * t_tiles, 8));
  hipLaunchKernelGGL((TileKernel<E, kN, kT, kWN, kWT, kStages>), dim3(grid), dim3(64 * kWN * kWT), 0, stream, g, n_tiles,
                     t_tiles, first);
}

template <typename E>
void LaunchAll(const LoraArgs& g, hipStream_t stream) {
  const uint64_t a_bytes = static_cast<uint64_t>(g.adapters) * g.max_rank * g.in_dim * sizeof(LowOf<E>);
  const uint64_t ranks = static_cast<uint64_t>(g.batch) * g.max_rank;
  // (A lane's offset into the adapters is 32 bits there.)
  if (g.a != nullptr && g.tokens <= kFewRows && ranks <= kFewRanks && a_bytes < (1ull << 31)) {
    hipLaunchKernelGGL((FewRowsKernel<E>), dim3(roost::CeilDiv(g.out_dim, 16)), dim3(64 * 12), 0, stream, g);
    return;
  }
  if (g.a != nullptr) {
    // Pieces of 64 rows read an adapter a fourth as often as pieces of 16, but are a fourth as many. Four sequences of 4096
    // channels to 64 outputs, by 16 and by 64, us a call: bf16, rank 16, 2,048 rows 17.7 and 20.6, 6,144 23.8 and 23.5, 15,000
    // 51 and 50; rank 64 22.1 and 26.9, 33.5 and 28.7, 78 and 56; e4m3, rank 16, 15.2 and 17.8, 18.9 and 18.7, 34 and 30; rank
    // 64 18.2 and 20.6, 31.9 and 25.5, 67 and 45. At 4,480 rows pieces of 64 already gain (rank 16 22.7 and 21.9, rank 64 32.7
    // and 27.8): the border is on the safe side of where they are even.
    if (g.tokens / g.batch >= 64 && g.tokens >= 6144) {
      LaunchShrinkOfRows<E, 4>(g, stream);
    } else {
      LaunchShrinkOfRows<E, 1>(g, stream);
    }
  }
  // Few rows: 16 outputs a workgroup while that is one workgroup a CU, else 32, for a second round costs more. 16 rows of 4096
  // channels: to 4096 outputs 16.7 us by 16 and 18.0 by 32, to 6144 22.4 and 18.8; 32 rows: 18.0 and 20.0, 25.4 and 21.1.
  const bool wide = roost::CeilDiv(g.out_dim, 16) > kCus;
  if (g.tokens <= 16) return wide ? LaunchProduct<E, 2, 1, 4, 2, 4>(g, stream) : LaunchProduct<E, 1, 1, 8, 1, 2>(g, stream);
  if (g.tokens <= 32) return wide ? LaunchProduct<E, 2, 2, 4, 4, 4>(g, stream) : LaunchProduct<E, 1, 2, 4, 2, 4>(g, stream);
  // More rows: the smallest tile whose workgroups are one round. In tiles of 32 outputs x 64 rows, of 80 x 64 and of 64 x 64 by
  // TileKernel: 128 rows, 4096 to 4096, 28, 37 and 43 us; 256 rows 41, 35 and 43 us; 1,072 rows, 2048 to 1024, 30, 20 and 28 us.
  if (roost::CeilDiv(g.out_dim, 32) * roost::CeilDiv(g.tokens, 64) <= kCus) return LaunchProduct<E, 2, 4, 4, 8, 3>(g, stream);
  if (roost::CeilDiv(g.out_dim, 80) * roost::CeilDiv(g.tokens, 64) <= kCus) return LaunchProduct<E, 5, 4, 4, 4, 2>(g, stream);
  if (g.tokens <= 64) return LaunchProduct<E, 2, 4, 4, 8, 3>(g, stream);
  // The adapters alone move an addend and an output: small tiles, many to a CU (4,480 rows of 4096 outputs, rank 16: 22 us,
  // by 256 x 256 36 us).
  if (g.w == nullptr) return LaunchTiles<E, 1, 2, 2, 1, 1>(g, 0, g.tokens, stream);
  // Tiles of many rows: a CU holds one workgroup of 256 x 256, 256 x 128 or 128 x 128, so they go in rounds of kCus, and a
  // larger tile's round does more for its time (4096 channels, bf16: about 116, 65 and 45 us). So the smallest tile with one
  // round, and 256 x 256 from where 256 x 128 would take a second one. 900 rows to 4096: 128 x 128 55, 64 x 64 73 us; 1,100 rows
  // to 4096: 256 x 128 75, 128 x 128 95, 64 x 64 87 us; 2,049 rows to 3,700 (255 of 256 x 128) 75, by 256 x 256 101 us; 2,304
  // rows to 4096 (288) 112, by 256 x 256 86 us; e4m3 70 and 48; 6,000 rows to 2048: 256 x 256 126, 128 x 128 153 us.
  const uint64_t across = roost::CeilDiv(g.out_dim, 256);
  const auto medium = [&](uint64_t rows) { return roost::CeilDiv(g.out_dim, 128) * roost::CeilDiv(rows, 128); };
  uint64_t done = 0;
  const uint64_t large = across * roost::CeilDiv(g.tokens, 256);
  if (across * roost::CeilDiv(g.tokens, 128) > kCus) {
    // Where the last round is a short one, the rows past the rounds before it take smaller tiles instead, if those are one
    // round: 4,400 rows to 4096 185 us against 225 in large tiles alone, 6,000 rows 220 against 235.
    done = (roost::CeilDiv(large, kCus) - 1) * kCus / across * 256;
    if (done == 0 || across * roost::CeilDiv(g.tokens - done, 128) > kCus) done = g.tokens;
    LaunchTiles<E, 2, 4, 4, 2, 2>(g, 0, done, stream);
    if (done == g.tokens) return;
  }
  if (medium(g.tokens - done) > kCus) return LaunchTiles<E, 2, 2, 4, 2, 3>(g, done, g.tokens, stream);
  if (done > 0 || medium(g.tokens) >= 128) return LaunchTiles<E, 2, 2, 2, 2, 4>(g, done, g.tokens, stream);
  return LaunchTiles<E, 1, 1, 2, 2, 4>(g, 0, g.tokens, stream);
}

}  // namespace

extern "C" ROOST_API RoostStatus roost_amd_gemm_lora_workspace(RoostContext* ctx, const void* params,
                                                               RoostWorkspaceSizes* sizes) {
  roost::Gate gate(kOp);
  gate.Expect(ctx != nullptr && sizes != nullptr, ROOST_STATUS_INVALID_ARGUMENT, "a context and a sizes record are required")
      .Header(params, sizeof(RoostAmdGemmLoraParams));
  ROOST_GATE_RETURN(gate);
  gate.Header(sizes, sizeof(RoostWorkspaceSizes));
  ROOST_GATE_RETURN(gate);
  const auto& p = *static_cast<const RoostAmdGemmLoraParams*>(params);
  return roost::CatchAll(kOp, [&]() -> RoostStatus {
    ROOST_RETURN_IF_FAILED(Admit(p, false));
    sizes->device_bytes = WorkspaceBytes(p);
    sizes->pinned_host_bytes = sizes->plan_bytes = 0;
    sizes->device_alignment = 256;
    return ROOST_STATUS_OK;
  });
}

extern "C" ROOST_API RoostStatus roost_amd_gemm_lora_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                                         void* stream) {
  roost::Gate gate(kOp);
  gate.Expect(ctx != nullptr, ROOST_STATUS_INVALID_ARGUMENT, "no context was passed")
      .Header(params, sizeof(RoostAmdGemmLoraParams));
  ROOST_GATE_RETURN(gate);
  const auto& p = *static_cast<const RoostAmdGemmLoraParams*>(params);
  return roost::CatchAll(kOp, [&]() -> RoostStatus {
    ROOST_RETURN_IF_FAILED(Admit(p, true));
    gate.Expect(roost::HasDeviceRegion(ws, WorkspaceBytes(p)), ROOST_STATUS_WORKSPACE_TOO_SMALL,
                "the call needs %llu bytes of 256-byte aligned device workspace",
                static_cast<unsigned long long>(WorkspaceBytes(p)));
    ROOST_GATE_RETURN(gate);
    if (p.tokens == 0 || p.batch == 0) return ROOST_STATUS_OK;
    ROOST_GATE_RETURN(roost::OnDevice(gate, ctx));
    LoraArgs g{};
    g.x = p.x.address, g.w = p.weight.address, g.a = p.lora_a.address, g.b = p.lora_b.address;
    g.x_scale = static_cast<const float*>(p.x_scale.address), g.w_scale = static_cast<const float*>(p.w_scale.address);
    g.lora_scale = static_cast<const float*>(p.lora_scale.address);
    g.ranks = static_cast<const int32_t*>(p.ranks.address), g.slots = static_cast<const int32_t*>(p.lora_slots.address);
    g.cu = static_cast<const int32_t*>(p.cu_seqlens.address);
    g.addend = p.addend.address, g.y = p.output.address;
    g.u = ws != nullptr ? static_cast<float*>(ws->device) : nullptr;
    g.u_part = LowRankElements(p);
    g.u_bf16 = reinterpret_cast<uint16_t*>(g.u + g.u_part);
    g.parts = LowRankParts(p);
    g.x_stride = Stride(p.x_stride, p.in_dim), g.addend_stride = Stride(p.addend_stride, p.out_dim);
    g.y_stride = Stride(p.output_stride, p.out_dim);
    g.tokens = p.tokens, g.batch = p.batch, g.in_dim = p.in_dim, g.out_dim = p.out_dim, g.adapters = p.adapters;
    g.max_rank = p.max_rank;
    g.addend_f32 = p.addend.dtype == ROOST_DTYPE_F32, g.y_f32 = p.output.dtype == ROOST_DTYPE_F32;
    const hipStream_t s = roost::Stream(stream);
    if (p.x.dtype == ROOST_DTYPE_F32) {
      LaunchAll<float>(g, s);
    } else if (p.x.dtype == ROOST_DTYPE_BF16) {
      LaunchAll<uint16_t>(g, s);
    } else if (g.y_f32) {
      LaunchAll<E4m3AsBf16>(g, s);
    } else {
      LaunchAll<E4m3>(g, s);
    }
    return roost::HipStatus(hipGetLastError(), kOp, "kernel launch");
  });
}
