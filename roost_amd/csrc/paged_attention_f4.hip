// PagedAttentionF4 for gfx950: attention over a KV cache held in 4 bits, decode rows and prompt chunks.
//
// Per query row (a token's head) with KV head h: s_j = scale q . k_j over the keys j that the row sees, p = softmax(s),
// out = sum_j p_j v_j, in one pass over the keys with a running maximum and sum. K and V come as e2m1 codes with a power of two
// for each 32 dims, and become bf16 exactly (v_cvt_scalef32_pk_bf16_fp4, two codes an instruction, the scale included), so the
// products are those of the bf16 matrix instructions with f32 sums. Each p is rounded to bf16 once in front of its product.

#include <cfloat>
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "cache_f4.h"

namespace {

using namespace roost_dev;

constexpr char kOp[] = "paged_attention_f4";
constexpr int32_t kMostKeys = 1 << 30;  // lengths are cut here, so that positions and their sums stay in 32 bits
constexpr float kGrow = 8.0f;           // the running maximum moves when a score is 2^8 above it

typedef float F4v __attribute__((ext_vector_type(4)));
typedef uint32_t U2 __attribute__((ext_vector_type(2)));
typedef uint32_t U4 __attribute__((ext_vector_type(4)));
typedef float F16v __attribute__((ext_vector_type(16)));
typedef short I4h __attribute__((ext_vector_type(4)));
typedef __bf16 B8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ F4v Mfma16(U4 a, U4 b, F4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(B8, a), __builtin_bit_cast(B8, b), c, 0, 0, 0);
}

__device__ __forceinline__ F16v Mfma32(U4 a, U4 b, F16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(B8, a), __builtin_bit_cast(B8, b), c, 0, 0, 0);
}

// cap tanh(s / cap) in log2 units, y the scaled score. What a kernel is built with:
//   kNearCap, caps up to 128: capl - 2 capl / (1 + 2^(k y)), off by at most 8 2^-23 cap whatever the score: 1.3e-4, below what
//     rounding p to bf16 makes of a score.
//   kFarCap, above: that would lose the score itself (0.02 at a cap of 1e5). With z = |y| / capl up to 1/4 y times a polynomial in
//     z^2, tanh(z) / z to 4e-9 (fitted for the least largest error), from there on as near: off by at most 16 2^-23 of the score.
//     A kernel of its own, for three times the instructions and more registers: a prompt chunk of 3,500 tokens on 500, 32 heads
//     over 8 of 128, takes 265 us, with a near cap 195, with none 142; a decode batch 133, 127 and 122.
enum Cap : int { kNoCap, kNearCap, kFarCap };
constexpr float kNearMost = 128.0f;  // the largest cap of kNearCap
struct SoftCap {
  float capl, k;  // k: 2 / cap, for kFarCap 1 / capl
};
template <int kCap>
__device__ __forceinline__ float Capped(float y, SoftCap c) {
  if constexpr (kCap == kNearCap) {
    return c.capl - 2.0f * c.capl * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y * c.k));
  } else {
    const float z = fabsf(y) * c.k, z2 = z * z;
    const float little = y * fmaf(z2, fmaf(z2, fmaf(z2, -0.05143305f, 0.13324264f), -0.33333242f), 1.0f);
    const float much = c.capl * fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * 2.88539008f)), 1.0f);
    return z <= 0.25f ? little : copysignf(much, y);
  }
}

struct Args {
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  roost::CacheF4View cache;
  const int32_t *cu, *tables, *lens, *indptr, *sequences;
  uint64_t q_stride, table_entries;
  uint32_t batch, tokens, q_heads, group, table_rows, max_blocks;
  float scale_log2;  // of the scores, times log2(e)
  SoftCap cap;
  uint32_t causal;
  int32_t window;
  // How the work is cut.
  float *part_o, *part_ml;   // the row kernel's partial rows: sums before division, and (maximum, sum)
  uint32_t *cut;             // what it tells its merge: all units, then those before each sequence; NULL: nothing is split
  uint32_t places;           // workgroups that share the units
  uint32_t max_units;        // of a sequence: all sequences' together, in all KV heads, stay below 2^32
  uint32_t short_tokens;     // sequences of at most so many tokens may be split
  uint32_t row_limit;        // the row kernel takes sequences of at most so many rows, the tile kernel the others
  float *tile_o, *tile_ml;   // the tile kernel's partial rows, in at most tile_splits parts of its keys
  uint32_t tile_splits;
};

// The sum over the lanes up to this one, by lane shifts within rows of 16 and two broadcasts over them.
__device__ __forceinline__ uint32_t WaveScan(uint32_t v) {
  const auto add = [&](uint32_t o) { v += o; };
  add(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x111, 0xf, 0xf, false)));
  add(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x112, 0xf, 0xf, false)));
  add(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x114, 0xf, 0xf, false)));
  add(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x118, 0xf, 0xf, false)));
  add(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x142, 0xa, 0xf, false)));
  add(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x143, 0xc, 0xf, false)));
  return v;
}
__device__ __forceinline__ uint32_t LaneOf(uint32_t v, int lane) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}
__device__ __forceinline__ uint32_t WaveSum(uint32_t v) { return LaneOf(WaveScan(v), 63); }

// ---- A sequence ---------------------------------------------------------------------------------------------------------

struct Sequence {
  int32_t first, count;   // tokens
  int32_t keys;
  int32_t blocks;         // its entries of the tables, from `entry` on
  int64_t entry;
};

// Lane `from`'s sequence.
__device__ __forceinline__ Sequence SequenceOfLane(const Sequence& s, int from) {
  const auto of = [&](int32_t v) { return __builtin_amdgcn_readlane(v, from); };
  Sequence t;
  t.first = of(s.first), t.count = of(s.count), t.keys = of(s.keys), t.blocks = of(s.blocks);
  t.entry = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(of(static_cast<int32_t>(s.entry)))) |
                                 static_cast<uint64_t>(static_cast<uint32_t>(of(static_cast<int32_t>(s.entry >> 32)))) << 32);
  return t;
}

__device__ __forceinline__ Sequence SequenceOf(const Args& a, uint32_t b) {
  Sequence s;
  const int32_t most = static_cast<int32_t>(a.tokens);
  s.first = min(max(a.cu[b], 0), most);
  s.count = min(max(a.cu[b + 1], s.first), most) - s.first;
  const uint32_t shift = a.cache.page_shift;
  int64_t keys = 0;
  s.blocks = 0;
  s.entry = 0;
  if (a.indptr != nullptr) {
    const int64_t begin = a.indptr[b], end = min(static_cast<int64_t>(a.indptr[b + 1]), static_cast<int64_t>(a.table_entries));
    if (begin >= 0 && end > begin) {
      s.blocks = static_cast<int32_t>(end - begin);
      s.entry = begin;
      keys = ((end - begin - 1) << shift) + min(max(a.lens[b], 0), 1 << shift);
    }
  } else {
    const int32_t row = a.sequences != nullptr ? a.sequences[b] : static_cast<int32_t>(b);
    if (static_cast<uint32_t>(row) < a.table_rows) {
      s.blocks = static_cast<int32_t>(a.max_blocks);
      s.entry = static_cast<int64_t>(row) * a.max_blocks;
      keys = min(static_cast<int64_t>(max(a.lens[row], 0)), static_cast<int64_t>(a.max_blocks) << shift);
    }
  }
  s.keys = static_cast<int32_t>(min(keys, static_cast<int64_t>(kMostKeys)));
  return s;
}

// The first key that any of the sequence's tokens from `token` on sees, down to a multiple of 16.
__device__ __forceinline__ int32_t FirstKey(const Args& a, const Sequence& s, int32_t token) {
  return a.window < 0 ? 0 : max(0, s.keys - s.count + token - a.window) & ~15;
}

constexpr int32_t kUnit = 128;            // keys: what the work of a batch is counted and cut in
constexpr uint32_t kMaxScheduled = 704;   // sequences of a batch whose keys may be split (their units' room in LDS)

// Whether the row kernel takes a sequence, and the units that its keys are (at most max_units: a last one takes what is left). 0:
// not its own. One unit where the sequence is not to be split.
__device__ __forceinline__ uint32_t UnitsOf(const Args& a, const Sequence& s) {
  const int64_t rows = static_cast<int64_t>(s.count) * a.group;
  if (rows == 0 || rows > static_cast<int64_t>(a.row_limit)) return 0;
  if (s.count > static_cast<int32_t>(a.short_tokens)) return 1;
  const int32_t units = (s.keys - FirstKey(a, s, 0) + kUnit - 1) / kUnit;
  return min(static_cast<uint32_t>(max(units, 1)), a.max_units);
}

// All units, sequence by sequence, in each KV head after KV head, dealt to `places` workgroups in turn, the first of them one
// more: the units of place c, and the place of unit x.
struct Deal {
  uint32_t each, more;  // more: places that have each + 1
  __device__ __forceinline__ Deal(uint32_t units, uint32_t places) : each(units / places), more(units - each * places) {}
  __device__ __forceinline__ uint32_t Begin(uint32_t c) const { return c * each + min(c, more); }
  __device__ __forceinline__ uint32_t PlaceOf(uint32_t x) const {
    const uint32_t longer = more * (each + 1);
    return x < longer ? x / (each + 1) : more + (x - longer) / each;
  }
};

// ---- The row kernel -----------------------------------------------------------------------------------------------------------
// Up to 16 kTiles rows (a few tokens' query heads of one KV head) against one part of a sequence's keys: decode. Bound by the
// cache's bytes, 1.06 D a key and KV head: 64 sequences of 500 to 16,000 keys, 32 heads over 8 of 128, 632 MB, take 128 us (4.9
// TB/s; a copy reaches 5.1, a stream that only reads 7.0) and the merge of their parts 6.
//
// Operands of v_mfma_f32_16x16x32_bf16, lane l = 16 g + m: A[m][8 g + j], B[8 g + j][m], result [4 g + i][m].
//   S^T = K Q^T: key m of 16 as A, query row m as B. The contraction runs over the dims in any order, so lane (m, g) takes its
//   key's 16 bytes g, dims 32 g .. 32 g + 31 (head_dim 128): one scale a lane, word s the operand of step s.
//   O^T = V^T P^T: dim as A, keys contracted. Lane (m, g) of S^T holds rows' scores of keys 4 g + i of both 16-key groups; as B
//   it needs eight keys: those. So keys are contracted in the order 16 (j / 4) + 4 g + j % 4, and p goes from result to operand
//   without leaving the lane. A's lane (m, g) takes dims D / 16 m .. of those eight keys: one word a key (head_dim 128), eight
//   dims a lane, dim d of the word the operand of product d.
//
// Four wavefronts take the part's steps of 32 keys in turn, each through a ring of its own in LDS that global_load_lds fills:
// 34 D bytes a step, kStages steps under way without a register, no barrier until the results meet. A step's copies are awaited
// by count.
//
// The units (128 keys of one KV head) of all sequences are dealt evenly to as many workgroups as the chip holds at once, each a
// run of them, whatever sequences and KV heads that run through: a sequence's length then costs what it reads and no
// workgroup waits for another. A KV head that a run holds whole is written out; of one that is cut, each workgroup leaves sums
// for the merge: a run is cut at its two ends at most, so two places a workgroup hold them. Every workgroup finds its run by itself
// from the lengths on the device, which a captured call cannot know before.
constexpr int kRowWaves = 4;
constexpr int kStep = 32;  // keys a wavefront takes at a time

template <int D>
struct RowRing {
  static constexpr int kCodes = kStep * D / 2;            // bytes of K's, and of V's, codes of a step
  static constexpr int kScales = 2 * D < 256 ? 256 : 2 * D;  // of both scales: [K, V][group][block][16 keys], at least one copy's
  static constexpr int kStage = 2 * kCodes + kScales;
  static constexpr int kCopies = 2 * kCodes / 1024 + kScales / 256;
  static constexpr int kStages = D == 256 ? 2 : 3;
};

// Workgroups of the row kernel that a CU holds, which its launch bounds ask for and the host deals the keys to. One tile of rows:
// 4, 3 and 2 at head_dim 64, 128 and 256, by LDS (29, 54 and 71 KB) and registers (128, 168 and 216); two tiles: 2, by registers
// (174 and 230). Dealt to more than it holds, a second round follows: 64 sequences of 5 tokens and 500 to 16,000 keys, 32 heads
// over 8 of 128, take 192 us, dealt to 3 a CU 206; a token of 32 heads a KV head 65 against 80.
constexpr uint32_t RowsResident(uint32_t d, uint32_t tiles) { return tiles == 2 || d == 256 ? 2 : d == 128 ? 3 : 4; }

// The memory that p points at in each lane to LDS, 16 (or 4) bytes a lane, one behind the other from `lds` on. M0 is read
// a wait state after its write.
__device__ __forceinline__ void Copy16(const void* p, uint32_t lds) {
  uint32_t m0;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(m0) : "v"(p), "s"(lds) : "memory");
}
// A byte a lane, each to a word of its own.
__device__ __forceinline__ void Copy1(const void* p, uint32_t lds) {
  uint32_t m0;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(m0) : "v"(p), "s"(lds) : "memory");
}
__device__ __forceinline__ void Copy4(const void* p, uint32_t lds) {
  uint32_t m0;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(m0) : "v"(p), "s"(lds) : "memory");
}

typedef __attribute__((address_space(3))) unsigned char LdsByte;
__device__ __forceinline__ uint32_t LdsAddress(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const LdsByte*)p));
}

template <int D, int kTiles, int kCap>
__global__ void __launch_bounds__(64 * kRowWaves, RowsResident(D, kTiles)) RowAttentionKernel(Args a) {
  typedef RowRing<D> Ring;
  constexpr int kWords = D / 32;   // of a lane's key
  constexpr int kDt = D / 16;      // dims of a lane's V word(s): products of 16 dims each
  constexpr int kBlocks = D / 32;
  constexpr int kStages = Ring::kStages;
  struct Result {
    float o[kRowWaves][16][D];
    float ml[kRowWaves][2][16];
  };
  constexpr int kBytes = kRowWaves * kStages * Ring::kStage;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[kBytes > sizeof(Result) ? kBytes : sizeof(Result)];
  Result& result = *reinterpret_cast<Result*>(lds);  // once all wavefronts are through with their rings

  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t heads = a.cache.kv_heads;
  __shared__ uint16_t units[kMaxScheduled];
  // Workgroup i runs on die i % 8: each die takes neighbouring runs, so that the scales of two heads, which share a line of
  // memory, come to one L2.
  const uint32_t share = (a.places + 7) / 8, place = blockIdx.x % 8 * share + blockIdx.x / 8;
  if (blockIdx.x / 8 >= share || place >= a.places) return;
  // The run [x, end) of units; the sequence of x, the units before it and its own.
  uint32_t x = 0, end = 0, before = 0, b = place / heads, own = 1;
  Sequence s;
  const auto find = [&](uint32_t mine) {  // mine: the units of sequence `lane`, for a batch of up to 64
    const uint32_t y = x / heads;
    uint32_t base = 0, sum = 0;
    for (;; base += 64) {
      const uint32_t here = a.batch <= 64 ? mine : base + lane < a.batch ? units[base + lane] : 0;
      const uint32_t to = sum + WaveScan(here);
      const uint64_t past = __ballot(y < to);
      if (past != 0) {
        const int at = __builtin_ctzll(past);
        b = base + static_cast<uint32_t>(at);
        own = LaneOf(here, at);
        before = LaneOf(to, at) - own;
        return;
      }
      sum = LaneOf(to, 63);
    }
  };
  uint32_t mine = 0;
  if (a.cut != nullptr) {
    uint32_t sum = 0;
    Sequence of{};
    if (a.batch <= 64) {
      if (lane < a.batch) of = SequenceOf(a, lane), mine = UnitsOf(a, of);
      sum = WaveSum(mine);
    } else {
      for (uint32_t i = threadIdx.x; i < a.batch; i += 64 * kRowWaves) {
        units[i] = static_cast<uint16_t>(UnitsOf(a, SequenceOf(a, i)));
      }
      __syncthreads();
      for (uint32_t i = lane; i < a.batch; i += 64) sum += units[i];
      sum = WaveSum(sum);
    }
    const Deal deal(sum * heads, a.places);
    x = deal.Begin(place), end = deal.Begin(place + 1);
    if (place == 0 && threadIdx.x == 0) a.cut[0] = sum;
    if (x >= end) return;
    find(mine);
    s = a.batch <= 64 ? SequenceOfLane(of, static_cast<int>(b)) : SequenceOf(a, b);
  } else {
    s = SequenceOf(a, b);
    if (UnitsOf(a, s) == 0) return;
  }

#pragma unroll 1
  for (bool opening = true;; opening = false) {
    // One KV head's part of the run.
    const uint32_t head = a.cut != nullptr ? (x - before * heads) / own : place % heads;
    const uint32_t from = a.cut != nullptr ? x - before * heads - head * own : 0;
    const uint32_t to = a.cut != nullptr ? min(own, from + (end - x)) : 1;
    const bool whole = from == 0 && to == own;
    const int32_t rows = s.count * static_cast<int32_t>(a.group);
    if (a.cut != nullptr && from == 0 && head == 0 && threadIdx.x == 0) a.cut[1 + b] = before;
    const int32_t k0 = FirstKey(a, s, 0) + static_cast<int32_t>(from) * kUnit;
    const int32_t k1 = to == own ? s.keys : k0 + static_cast<int32_t>(to - from) * kUnit;

    const int32_t steps = max(0, (k1 - k0 + kStep - 1) / kStep), my_steps = (steps + kRowWaves - 1 - w) / kRowWaves;
    const auto key_of = [&](int32_t step) { return k0 + (step * kRowWaves + w) * kStep; };
    const uint32_t shift = a.cache.page_shift, in_page = (1u << shift) - 1;
    unsigned char* const ring = lds + w * kStages * Ring::kStage;

    // Page ids of a window of 32 steps, a group of 16 keys a lane; -1 for a page that is none.
    const auto ids_of = [&](int32_t window) {
      const int32_t key = key_of(window * 32 + lane / 2) + 16 * (lane & 1), at = key >> shift;
      int32_t id = -1;
      if (key < k1 && at < s.blocks) id = a.tables[s.entry + at];
      return static_cast<uint32_t>(id) < a.cache.pages ? id : -1;
    };

    // One step's codes and scales to the ring. Pages that are none: page 0, whose keys are masked.
    const auto issue = [&](int32_t step, int32_t ids) {
      const uint32_t to = LdsAddress(ring) + static_cast<uint32_t>(step % kStages) * Ring::kStage;
      uint64_t row[2], scale_row[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int32_t id = __builtin_amdgcn_readlane(ids, (2 * step + t) & 63);
        const uint32_t key = static_cast<uint32_t>(key_of(step) + 16 * t) & in_page;
        const uint64_t head_page = static_cast<uint64_t>(max(id, 0)) * a.cache.kv_heads + head;
        row[t] = ((head_page << shift) + key) * (D / 2);
        scale_row[t] = ((head_page * kBlocks) << shift) + key;
      }
#pragma unroll
      for (int i = 0; i < Ring::kCodes / 1024; ++i) {
        const uint32_t byte = 1024 * i + 16 * lane;  // of [group][16 keys x D / 2]
        const uint64_t from = (D == 64 ? (lane < 32 ? row[0] : row[1]) : row[i / (D / 128)]) + byte % (8 * D);
        Copy16(a.cache.k + from, to + 1024 * i);
        Copy16(a.cache.v + from, to + Ring::kCodes + 1024 * i);
      }
#pragma unroll
      for (int i = 0; i < Ring::kScales / 256; ++i) {
        const uint32_t x = 64 * i + lane, block = x / 4 % kBlocks, t = x / (4 * kBlocks) % 2, value = x / (8 * kBlocks) % 2;
        const uint64_t from = (t == 0 ? scale_row[0] : scale_row[1]) + (block << shift) + 4 * (x % 4);
        Copy4((value ? a.cache.v_scales : a.cache.k_scales) + from, to + 2 * Ring::kCodes + 256 * i);
      }
    };

    for (int32_t tile = 0; tile * 16 * kTiles < rows; ++tile) {
      // Query rows: lane m's of each 16.
      int32_t pos[kTiles];
      U4 q[kTiles][kWords];
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        const int32_t r = (tile * kTiles + n) * 16 + m;
        const bool ok = r < rows;
        const int32_t token = ok ? r / static_cast<int32_t>(a.group) : 0;
        const uint32_t h = head * a.group + (ok ? r - token * static_cast<int32_t>(a.group) : 0);
        pos[n] = ok ? s.keys - s.count + token : -1;
        const uint16_t* qr = a.q + static_cast<uint64_t>(s.first + token) * a.q_stride + static_cast<uint64_t>(h) * D;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          const int d = D == 64 ? 16 * g + 8 * i : 128 * (i / 4) + 32 * g + 8 * (i % 4);
          const U4 x = *reinterpret_cast<const U4*>(qr + d);
          q[n][i] = ok ? x : U4{0, 0, 0, 0};
        }
      }

      F4v o[kTiles][kDt];
      float top[kTiles], sum[kTiles];
      // careful: a block of V that is NaN multiplies as zeros, and makes the outputs of the rows that see it NaN by hand; without,
      // its NaN would reach the rows that do not see it as well. Only taken where a first pass left a NaN.
      const auto pass = [&](bool careful) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          top[n] = -INFINITY, sum[n] = 0.0f;
#pragma unroll
          for (int d = 0; d < kDt; ++d) o[n][d] = F4v{0, 0, 0, 0};
        }
        int32_t ids = ids_of(0), ids_next = my_steps > 32 ? ids_of(1) : -1;
        uint64_t bad_issued = __ballot(ids < 0), bad = bad_issued;  // groups without a page: of the window issued from, of this one
#pragma unroll
        for (int i = 0; i < kStages; ++i) {
          if (i < my_steps) issue(i, ids);
        }
#pragma unroll 1
        for (int32_t step = 0; step < my_steps; ++step) {
          if ((step & 31) == 0) bad = bad_issued;
          if (step + kStages <= my_steps) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kStages - 1) * Ring::kCopies) : "memory");
          } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          }
          // The lane's share of the step: key m's codes and scales in each group, its dims of the eight keys and their scales.
          uint32_t kc[2][kWords], ks[2][D == 256 ? 2 : 1], vc[8][D == 256 ? 2 : 1], vs[2];
          {
            const unsigned char* at = ring + static_cast<uint32_t>(step % kStages) * Ring::kStage;
            const unsigned char* sc = at + 2 * Ring::kCodes;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if constexpr (D == 64) {
                const U2 x = *reinterpret_cast<const U2*>(at + 512 * t + 32 * m + 8 * g);
                kc[t][0] = x[0], kc[t][1] = x[1];
                ks[t][0] = sc[16 * (t * kBlocks + g / 2) + m];
              } else {
#pragma unroll
                for (int h = 0; h < D / 128; ++h) {
                  const U4 x = *reinterpret_cast<const U4*>(at + 8 * D * t + m * (D / 2) + 64 * h + 16 * g);
#pragma unroll
                  for (int i = 0; i < 4; ++i) kc[t][4 * h + i] = x[i];
                  ks[t][h] = sc[16 * (t * kBlocks + 4 * h + g) + m];
                }
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const unsigned char* p = at + Ring::kCodes + 8 * D * t + (4 * g + i) * (D / 2) + m * (D / 32);
                if constexpr (D == 64) {
                  vc[4 * t + i][0] = *reinterpret_cast<const uint16_t*>(p);
                } else if constexpr (D == 128) {
                  vc[4 * t + i][0] = *reinterpret_cast<const uint32_t*>(p);
                } else {
                  const U2 x = *reinterpret_cast<const U2*>(p);
                  vc[4 * t + i][0] = x[0], vc[4 * t + i][1] = x[1];
                }
              }
              vs[t] = *reinterpret_cast<const uint32_t*>(sc + 32 * kBlocks + 16 * (t * kBlocks + m / (512 / D)) + 4 * g);
            }
          }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read: the next copies may take the stage
          if (step + kStages < my_steps) {
            const int32_t next = step + kStages;
            if ((next & 31) == 0) {
              ids = ids_next;
              bad_issued = __ballot(ids < 0);
              if (next + 32 < my_steps) ids_next = ids_of(next / 32 + 1);
            }
            issue(next, ids);
          }

          const int32_t key0 = key_of(step);
          const uint32_t none = static_cast<uint32_t>(bad >> ((2 * step) & 63)) & 3;  // groups without a page
          const bool edge = key0 + kStep > k1 || none != 0;
          const bool mask = edge || (a.causal && key0 + kStep > s.keys - s.count + 1) ||
                            (a.window >= 0 && key0 < s.keys - 1 - a.window);
          const auto absent = [&](int t, int i) {  // key 16 t + 4 g + i is none of the part's
            return key0 + 16 * t + 4 * g + i >= k1 || (none >> t & 1) != 0;
          };
          F4v sc[kTiles][2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int n = 0; n < kTiles; ++n) sc[n][t] = F4v{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
              const float scale = F4Scale(ks[t][D == 256 ? i / 4 : 0]);
              const uint32_t c = kc[t][i];
              const U4 kk{FromF4<0>(c, scale), FromF4<1>(c, scale), FromF4<2>(c, scale), FromF4<3>(c, scale)};
#pragma unroll
              for (int n = 0; n < kTiles; ++n) sc[n][t] = Mfma16(kk, q[n][i], sc[n][t]);
            }
          }
          uint32_t nan_keys = 0;
          if (edge || careful) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t byte = vs[t] >> (8 * i) & 0xFF;
                const bool nan = careful && byte > kF4ByteHigh;
                const bool off = absent(t, i);
                if (nan && !off) nan_keys |= 1u << (4 * t + i);
                if (nan || off) vs[t] = (vs[t] & ~(0xFFu << (8 * i))) | 127u << (8 * i);  // finite, times p = 0
              }
            }
          }
          U4 p[kTiles];
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              y[j] = sc[n][j / 4][j % 4];
              if constexpr (kCap != kNoCap) y[j] = Capped<kCap>(y[j] * a.scale_log2, a.cap);
            }
            if (mask) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const int32_t key = key0 + 16 * (j / 4) + 4 * g + j % 4;
                const bool off = absent(j / 4, j % 4) | ((a.causal != 0) & (key > pos[n])) |
                                 ((a.window >= 0) & (key < pos[n] - a.window));
                y[j] = off ? -INFINITY : y[j];
              }
            }
            const float scale = kCap != kNoCap ? 1.0f : a.scale_log2;  // positive: the largest score stays the largest
            float mx = y[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) mx = fmaxf(mx, y[j]);
            mx *= scale;
            if (__any(mx > top[n] + kGrow)) {
              mx = fmaxf(mx, __shfl_xor(mx, 16));
              mx = fmaxf(mx, __shfl_xor(mx, 32));
              const float now = mx > top[n] ? mx : top[n];
              const float by = top[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top[n] - now);
              sum[n] *= by;
#pragma unroll
              for (int d = 0; d < kDt; ++d) o[n][d] *= by;
              top[n] = now;
            }
            const float base = top[n] == -INFINITY ? 0.0f : top[n];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              y[j] = __builtin_amdgcn_exp2f(fmaf(y[j], scale, -base));
              sum[n] += y[j];
            }
            p[n] = U4{PackBf16Rne(y[0], y[1]), PackBf16Rne(y[2], y[3]), PackBf16Rne(y[4], y[5]), PackBf16Rne(y[6], y[7])};
          }
          // Two dims of eight keys, then each dim's eight keys.
          const auto two = [&](auto pair, int word, int out) {
            uint32_t c[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              c[j] = FromF4<decltype(pair)::value>(vc[j][word], F4Scale(vs[j / 4] >> (8 * (j % 4)) & 0xFF));
            }
            U4 lo, hi;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              lo[j] = __builtin_amdgcn_perm(c[2 * j + 1], c[2 * j], 0x05040100u);
              hi[j] = __builtin_amdgcn_perm(c[2 * j + 1], c[2 * j], 0x07060302u);
            }
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
              o[n][out] = Mfma16(lo, p[n], o[n][out]);
              o[n][out + 1] = Mfma16(hi, p[n], o[n][out + 1]);
            }
          };
#pragma unroll
          for (int word = 0; word < (D == 256 ? 2 : 1); ++word) {
            two(std::integral_constant<int, 0>{}, word, 8 * word);
            two(std::integral_constant<int, 1>{}, word, 8 * word + 2);
            if constexpr (D > 64) {
              two(std::integral_constant<int, 2>{}, word, 8 * word + 4);
              two(std::integral_constant<int, 3>{}, word, 8 * word + 6);
            }
          }
          if (careful) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              for (uint64_t lanes = __ballot(nan_keys >> j & 1); lanes != 0; lanes &= lanes - 1) {
                const int from = __builtin_ctzll(lanes);  // dims D / 16 (from % 16) .. of a key of its group
                const int32_t key = key0 + 16 * (j / 4) + 4 * (from >> 4) + j % 4;
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
                  if ((a.causal && key > pos[n]) || (a.window >= 0 && key < pos[n] - a.window)) continue;
#pragma unroll
                  for (int d = 0; d < kDt; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                      if (4 * g + i == (from & 15)) o[n][d][i] = NAN;
                    }
                }
              }
            }
          }
        }
      };
      bool careful = false;
#pragma unroll 1
      for (;;) {
        pass(careful);
        if (careful) break;
        bool nan = false;
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int d = 0; d < kDt; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) nan |= o[n][d][i] != o[n][d][i];
        if (!__any(nan)) break;
        careful = true;
      }

      // The four wavefronts' results meet, 16 rows at a time.
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        const int32_t row0 = (tile * kTiles + n) * 16;
        float l = sum[n];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        __syncthreads();  // the rings, or the rows before, are read
        if (g == 0) result.ml[w][0][m] = top[n], result.ml[w][1][m] = l;
        if (row0 + m < rows) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < kDt; d += 4) {
              *reinterpret_cast<F4v*>(&result.o[w][m][(4 * g + i) * kDt + d]) =
                  F4v{o[n][d][i], o[n][d + 1][i], o[n][d + 2][i], o[n][d + 3][i]};
            }
        }
        __syncthreads();
        constexpr int kThreadsPerRow = 16, kPer = D / kThreadsPerRow;  // 16 rows x 16 threads
        const int r = threadIdx.x / kThreadsPerRow, d0 = (threadIdx.x % kThreadsPerRow) * kPer;
        const int32_t row = row0 + r;
        if (row >= rows) continue;
        float big = result.ml[0][0][r];
#pragma unroll
        for (int x = 1; x < kRowWaves; ++x) big = fmaxf(big, result.ml[x][0][r]);
        float total = 0.0f, f[kRowWaves], y[kPer];
#pragma unroll
        for (int x = 0; x < kRowWaves; ++x) {
          f[x] = result.ml[x][0][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(result.ml[x][0][r] - big);
          total += result.ml[x][1][r] * f[x];
        }
#pragma unroll
        for (int d = 0; d < kPer; ++d) {
          y[d] = 0.0f;
#pragma unroll
          for (int x = 0; x < kRowWaves; ++x) y[d] += result.o[x][r][d0 + d] * f[x];
        }
        const int32_t token = row / static_cast<int32_t>(a.group);
        const uint32_t h = head * a.group + static_cast<uint32_t>(row - token * static_cast<int32_t>(a.group));
        if (!whole) {
          // A part that began in an earlier run opens this one; else it goes on in the next.
          const uint64_t at = (2 * static_cast<uint64_t>(place) + (opening && from != 0 ? 0 : 1)) * a.short_tokens * a.group +
                              static_cast<uint32_t>(row);
#pragma unroll
          for (int d = 0; d < kPer; d += 4) {
            *reinterpret_cast<F4v*>(a.part_o + at * D + d0 + d) = F4v{y[d], y[d + 1], y[d + 2], y[d + 3]};
          }
          if (d0 == 0) a.part_ml[2 * at] = big, a.part_ml[2 * at + 1] = total;
        } else {
          const float inv = total > 0.0f ? 1.0f / total : total == total ? 0.0f : NAN;
          const uint64_t at = static_cast<uint64_t>(s.first + token) * a.q_heads + h;
#pragma unroll
          for (int d = 0; d < kPer; d += 4) {
            *reinterpret_cast<U2*>(a.out + at * D + d0 + d) = U2{PackBf16Rne(y[d] * inv, y[d + 1] * inv),
                                                                 PackBf16Rne(y[d + 2] * inv, y[d + 3] * inv)};
        }
        if (a.lse != nullptr && d0 == 0) {
          a.lse[at] = total > 0.0f ? big + __builtin_amdgcn_logf(total) : total == total ? -INFINITY : NAN;
        }
        }
      }
      __syncthreads();  // the results are read: the rings may be filled again
    }
    x += to - from;
    if (x >= end) return;
    if (x >= (before + own) * heads) {
      find(mine);
      s = SequenceOf(a, b = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(b))));
    }
  }
}

// ---- The tile kernel ----------------------------------------------------------------------------------------------------------
// 256 rows of one sequence and KV head (rows are its tokens' query heads, token by token) against the keys that they see, 64 or
// 128 at a time: prompt chunks. Bound by the matrix instructions and, beside them, by the softmax and LDS reads: 1.0 PFLOP/s over
// two prompts of 3,500 to 4,096 tokens on prefixes, 32 heads over 8 of 128.
//
// A tile's codes go to LDS as bf16 once for all wavefronts, a lane a block of 32 dims (16 bytes, one scale): 16 conversions a lane
// for 64 keys at head_dim 128, where converting in each wavefront would take 128. Codes of the next tile are under way
// during a tile's products, straight into LDS, where each lane finds its own again: held in registers they would not fit beside
// 32 rows' queries and sums at head_dim 256. LDS holds two converted tiles, so there is one barrier a tile.
//
// v_mfma_f32_32x32x16_bf16, lane l = 32 g + m: A[m][8 g + j], B[8 g + j][m], result register v at [8 (v / 4) + 4 g + v % 4][m].
//   S^T = K Q^T with 32 keys as A and the wavefront's 32 rows as B. A lane then holds, of its row, keys 4 g + i of each 8; the
//   products O^T = V^T P^T contract the keys in that order, so p stays in its lane, and V^T's operand (dim m, four keys twice) is
//   read from LDS by transposing reads.
// LDS: reads of 16 bytes a lane want 16 rows' pieces apart in 256 bytes, the converted codes' stores eight lanes' apart in 128
// (counted: eight lanes a cycle). K rows are padded by 16 bytes for the first; V's 64-byte chunks change places by the key for the
// transposing reads of four keys x 64 bytes. The stores' eight lanes have 8 / (D / 32) keys, so pieces change places by what those
// bits do not tell apart: no conflict is left (28% of the LDS cycles at head_dim 128 before; 5% of the time).

constexpr int kTileWaves = 8;
constexpr int kTileKeys = 64;  // what a tile's keys are cut into parts by

__device__ __forceinline__ U2 LdsTranspose(const unsigned char* base, uint32_t off) {
  auto* p = reinterpret_cast<__attribute__((address_space(3))) I4h*>(const_cast<LdsByte*>((const LdsByte*)base + off));
  return __builtin_bit_cast(U2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
}

template <int D, int kKeys, int kPieces>
struct TileLds {
  static constexpr int kKeyRow = 2 * D + 16;
  unsigned char k[2][kKeys * kKeyRow];
  unsigned char v[2][kKeys * 2 * D];
  U4 codes[kTileWaves][kPieces][64];        // of the next tile, a block a lane
  uint32_t scales[kTileWaves][kPieces][64];
  uint32_t bad[3];                // groups of 16 keys without a page, of this tile, the next and the one after
  uint32_t nan[3][kKeys];     // blocks of V that are NaN; only kept in a careful pass
};

// Where block `block`, piece `piece` (8 dims) of a key lies in LDS, V's and K's, and how V's pieces change places.
template <int D>
constexpr uint32_t SwapOf(uint32_t key, uint32_t block) {
  return D == 64 ? key & 3 : D == 128 ? ((key ^ key >> 2) & 3) ^ (block & 2) : block >> 1;
}
template <int D>
__device__ __forceinline__ uint32_t ValueAt(uint32_t key, uint32_t block, uint32_t piece) {
  const uint32_t swap = D == 64 ? key >> 1 & 1 : key & 3;
  return key * 2 * D + ((block ^ swap) * 64) + ((piece ^ SwapOf<D>(key, block)) * 16);
}
template <int D>
__device__ __forceinline__ uint32_t KeyAt(uint32_t key, uint32_t block, uint32_t piece) {
  return key * (2 * D + 16) + 64 * block + 16 * (D == 64 ? piece : piece ^ (block & 2)) + (D == 256 ? 16 * (block >> 2) : 0);
}

// Tile `rank` of all sequences' that have more rows than row_limit; a sequence's last tiles first, whose rows see most keys.
// Every wavefront finds it by itself.
__device__ __forceinline__ bool FindTile(const Args& a, uint32_t rank, uint32_t rows_a_tile, uint32_t& b, int32_t& tile) {
  const int lane = threadIdx.x & 63;
  const int32_t most = static_cast<int32_t>(a.tokens);
  for (uint32_t base = 0; base < a.batch; base += 64) {
    uint32_t tiles = 0;
    if (base + lane < a.batch) {
      const int32_t first = min(max(a.cu[base + lane], 0), most);
      const uint32_t rows = static_cast<uint32_t>(min(max(a.cu[base + lane + 1], first), most) - first) * a.group;
      tiles = rows > a.row_limit ? (rows + rows_a_tile - 1) / rows_a_tile : 0;
    }
    const uint32_t end = WaveScan(tiles);
    const uint64_t here = __ballot(rank < end);
    if (here != 0) {
      const int at = __builtin_ctzll(here);
      b = base + static_cast<uint32_t>(at);
      tile = static_cast<int32_t>(LaneOf(end, at)) - 1 - static_cast<int32_t>(rank);
      return true;
    }
    rank -= LaneOf(end, 63);
  }
  return false;
}

// A tile's keys, and their parts.
struct TileKeys {
  int32_t begin, end, part;
  uint32_t parts;
};
__device__ __forceinline__ TileKeys KeysOfTile(const Args& a, const Sequence& s, int32_t tile, int32_t rows_a_tile) {
  const int32_t group = static_cast<int32_t>(a.group);
  const int32_t first = tile * rows_a_tile / group, last = min((tile * rows_a_tile + rows_a_tile - 1) / group, s.count - 1);
  TileKeys k;
  k.begin = FirstKey(a, s, first);
  k.end = a.causal ? max(0, s.keys - s.count + last + 1) : s.keys;
  const int32_t n = max(0, k.end - k.begin);
  k.part = ((n + static_cast<int32_t>(a.tile_splits) - 1) / static_cast<int32_t>(a.tile_splits) + kTileKeys - 1) & ~(kTileKeys - 1);
  k.parts = n == 0 ? 1 : static_cast<uint32_t>((n + k.part - 1) / k.part);
  return k;
}

template <int D, int kCap>
__global__ void __launch_bounds__(64 * kTileWaves, kTileWaves / 4) TileAttentionKernel(Args a) {
  constexpr int kThreads = 64 * kTileWaves, kRows = 32 * kTileWaves;
  constexpr int kKs = D / 16, kDt = D / 32;
  constexpr int kHalves = D == 64 ? 2 : 1;  // of a tile's keys that are scored together (at 128 the registers of two cost 1%)
  // Keys at a time: as many as LDS holds twice, two workgroups' at head_dim 64. 128 instead of 64, half the barriers: 606 -> 566 us
  // for two prompts of 3,500 to 4,096 tokens on prefixes at 128, 166 -> 147 for four of 2,000 to 4,000; 96 -> 92 for four of 1,000
  // to 2,000 at 64.
  constexpr int kKeys = D == 256 ? 64 : 128;
  constexpr int kBlocks = kKeys * D / 32;     // of K's, and of V's, of a tile
  constexpr int kPieces = (2 * kBlocks + kThreads - 1) / kThreads;  // blocks of 32 codes that a lane stages
  typedef TileLds<D, kKeys, kPieces> Lds;
  __shared__ __attribute__((aligned(16))) Lds lds;

  const uint32_t head = blockIdx.x % a.cache.kv_heads, split = blockIdx.x / a.cache.kv_heads % a.tile_splits;
  uint32_t b = 0;
  int32_t tile = 0;
  if (!FindTile(a, blockIdx.x / a.cache.kv_heads / a.tile_splits, kRows, b, tile)) return;
  b = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(b)));
  tile = __builtin_amdgcn_readfirstlane(tile);
  const Sequence s = SequenceOf(a, b);
  const TileKeys range = KeysOfTile(a, s, tile, kRows);
  if (split >= range.parts) return;
  const int32_t k0 = range.begin + static_cast<int32_t>(split) * range.part;
  const int32_t k1 = min(range.end, k0 + range.part);
  const int32_t tiles = k1 > k0 ? (k1 - k0 + kKeys - 1) / kKeys : 0;

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t group = static_cast<int32_t>(a.group), rows = s.count * group;
  const int32_t before = s.keys - s.count;  // the first token's position
  // Lane `id`'s row: its token, -1 where there is none, and its query head.
  const auto row_of = [&](int id, int32_t& token, uint32_t& h) {
    const int32_t r = tile * kRows + 32 * w + (id & 31);
    token = r < rows ? r / group : -1;
    h = head * a.group + static_cast<uint32_t>(r < rows ? r - token * group : 0);
  };
  // Positions of the wavefront's first and last row.
  const int32_t low = before + (tile * kRows + 32 * w) / group;
  const int32_t high = before + min((tile * kRows + 32 * w + 31) / group, s.count - 1);
  const int32_t last = a.causal ? min(high, k1 - 1) : k1 - 1;  // the last key of the part that its rows see
  const bool idle = tile * kRows + 32 * w >= rows;  // the wavefront has no row, and only stages

  U4 q[kKs];
  {
    int32_t token;
    uint32_t h;
    row_of(tid, token, h);
    const uint16_t* qr = a.q + static_cast<uint64_t>(s.first + max(token, 0)) * a.q_stride + static_cast<uint64_t>(h) * D + 8 * g;
#pragma unroll
    for (int i = 0; i < kKs; ++i) {
      const U4 x = *reinterpret_cast<const U4*>(qr + 16 * i);
      q[i] = token >= 0 ? x : U4{0, 0, 0, 0};
    }
  }

  // Staging: piece tid + i kThreads of [K, V] x 64 keys x blocks. From head_dim 128 on a wavefront's 64 pieces are of one page.
  const uint32_t shift = a.cache.page_shift, in_page = (1u << shift) - 1;
  const auto piece_of = [&](int i, int id, bool& value, int32_t& key, uint32_t& block) {
    const int p = id + i * kThreads;
    value = p >= kBlocks;
    key = (p & (kBlocks - 1)) / (D / 32);
    block = static_cast<uint32_t>(p) & (D / 32 - 1);
    return p < 2 * kBlocks;
  };
  int32_t ids[kPieces];
  uint32_t none = 0;  // pieces of the tile under way that have no page
  const auto load_ids = [&](int32_t t, int id) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      bool value;
      int32_t key;
      uint32_t block;
      ids[i] = -1;
      if (!piece_of(i, id, value, key, block) || t >= tiles) continue;
      const int32_t k = k0 + t * kKeys + key, entry = k >> shift;
      if ((k & ~15) < k1 && entry < s.blocks) ids[i] = a.tables[s.entry + entry];
    }
  };
  const auto load_codes = [&](int32_t t, int id) {
    none = 0;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      bool value;
      int32_t key;
      uint32_t block;
      if (!piece_of(i, id, value, key, block)) continue;
      int32_t page = D == 64 ? ids[i] : __builtin_amdgcn_readfirstlane(ids[i]);
      if (static_cast<uint32_t>(page) >= a.cache.pages) none |= 1u << i, page = 0;  // masked: any codes will do
      const uint32_t within = static_cast<uint32_t>(k0 + t * kKeys + key) & in_page;
      const uint64_t head_page = static_cast<uint64_t>(page) * a.cache.kv_heads + head;
      Copy16((value ? a.cache.v : a.cache.k) + ((head_page << shift) + within) * (D / 2) + 16 * block, LdsAddress(lds.codes[w][i]));
      Copy1((value ? a.cache.v_scales : a.cache.k_scales) + ((head_page * (D / 32) + block) << shift) + within,
            LdsAddress(lds.scales[w][i]));
    }
  };
  const auto store = [&](int32_t t, int id, bool careful) {
    const int slot = t % 3;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      bool value;
      int32_t key;
      uint32_t block;
      if (!piece_of(i, id, value, key, block)) continue;
      if ((none >> i & 1) && block == 0) atomicOr(&lds.bad[slot], 1u << (key / 16));
      const U4 codes = lds.codes[w][i][id & 63];
      uint32_t byte = lds.scales[w][i][id & 63];
      if (value) {
        if ((none >> i & 1) || k0 + t * kKeys + key >= k1) byte = 127;  // whatever lies there: finite, times p = 0
        if (careful && byte > kF4ByteHigh) {
          byte = 127;
          atomicOr(&lds.nan[slot][key], 1u << block);
        }
      }
      const float scale = F4Scale(byte);
      unsigned char* const to = value ? lds.v[t & 1] : lds.k[t & 1];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t c = codes[j];
        const U4 x{FromF4<0>(c, scale), FromF4<1>(c, scale), FromF4<2>(c, scale), FromF4<3>(c, scale)};
        const uint32_t off = value ? ValueAt<D>(key, block, j) : KeyAt<D>(key, block, j);
        *reinterpret_cast<U4*>(to + off) = x;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read: the next codes may come
  };

  F16v o[kDt];
  float top, sum;
  const auto pass = [&](bool careful) {
    top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int d = 0; d < kDt; ++d)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[d][v] = 0.0f;
    if (tid < 3) lds.bad[tid] = 0;
    if (careful && tid < kKeys) lds.nan[0][tid] = lds.nan[1][tid] = lds.nan[2][tid] = 0;
    __syncthreads();
    if (tiles > 0) {
      load_ids(0, tid);
      load_codes(0, tid);
      load_ids(1, tid);
      store(0, tid, careful);
    }
#pragma unroll 1
    for (int32_t t = 0; t < tiles; ++t) {
      __syncthreads();  // tile t is in LDS; nobody reads tile t - 1 any more
      const int slot = t % 3, after = (t + 2) % 3;
      // What depends on the lane is made anew from its number each time: kept, it would at 64 leave room for one workgroup a CU
      // instead of two (four prompts of 1,000 to 2,000 tokens on prefixes, 32 heads over 8: 105 us, kept 125). At 128 there is
      // room, and it is kept (544 us; anew 620). At 256 all 256 registers are taken and 10 more values go to scratch (kept: 51):
      // in front of and behind this loop and in a careful pass; with a cap a query operand's four are read in it too.
      int tid = threadIdx.x;
      if constexpr (D != 128) asm volatile("" : "+v"(tid));
      const int lane = tid & 63, m = lane & 31, g = lane >> 5;
      if (tid == 0) lds.bad[after] = 0;
      if (careful && tid < kKeys) lds.nan[after][tid] = 0;
      if (t + 1 < tiles) {
        load_codes(t + 1, tid);
        load_ids(t + 2, tid);
      }
      const int32_t kb = k0 + t * kKeys;
      if (!idle && kb <= last) {
        const uint32_t bad = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(lds.bad[slot])));
        const bool mask = kb + kKeys > k1 || (a.causal && kb + kKeys - 1 > low) || bad != 0 ||
                          (a.window >= 0 && kb < high - a.window);
        const unsigned char* kt = lds.k[t & 1] + m * Lds::kKeyRow + 16 * g;
        const unsigned char* vt = lds.v[t & 1];
        // The transposing read of four keys x 16 dims by 16 lanes: lane 16 c + j addresses key j / 4, dims 4 (j % 4) of it.
        const uint32_t j = lane & 15, key4 = 4 * g + j / 4, piece = 2 * (lane >> 4 & 1) + (j % 4) / 2;
        uint32_t va[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) va[f] = ValueAt<D>(key4 + 8 * f, 0, piece) + 8 * (j & 1);
#pragma unroll (D == 256 ? 1 : kKeys / 32)  // at 256, by 3% faster so: fewer registers are kept over both halves
        for (int half = 0; half < kKeys / 32; half += kHalves) {
          if (half > 0 && kb + 32 * half > last) break;
          F16v sc[kHalves];
#pragma unroll
          for (int x = 0; x < kHalves; ++x)
#pragma unroll
            for (int v = 0; v < 16; ++v) sc[x][v] = 0.0f;
          // Operands are read two steps ahead of the products that use them: left alone, the compiler waits out every read in front
          // of its product at this number of registers. The same for V below.
          const unsigned char* kr = kt + 32 * half * Lds::kKeyRow;
          constexpr int kAhead = 2;
          U4 ka[kAhead][kHalves];
          const auto key = [&](int i, int x) {  // dims 16 i + 8 g .. of the lane's key
            return *reinterpret_cast<const U4*>(kr + 32 * x * Lds::kKeyRow + KeyAt<D>(0, i / 2, 2 * (i % 2)));
          };
#pragma unroll
          for (int i = 0; i < kAhead; ++i)
#pragma unroll
            for (int x = 0; x < kHalves; ++x) ka[i][x] = key(i, x);
#pragma unroll
          for (int i = 0; i < kKs; ++i)
#pragma unroll
            for (int x = 0; x < kHalves; ++x) {
              const U4 k = ka[i % kAhead][x];
              if (i + kAhead < kKs) ka[i % kAhead][x] = key(i + kAhead, x);
              sc[x] = Mfma32(k, q[i], sc[x]);
            }
          __builtin_amdgcn_sched_group_barrier(0x100, kAhead * kHalves, 0);
#pragma unroll
          for (int i = 0; i < (kKs - kAhead) * kHalves; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          }
          __builtin_amdgcn_sched_group_barrier(0x008, kAhead * kHalves, 0);
          if constexpr (kCap != kNoCap) {
#pragma unroll
            for (int x = 0; x < kHalves; ++x)
#pragma unroll
              for (int v = 0; v < 16; ++v) sc[x][v] = Capped<kCap>(sc[x][v] * a.scale_log2, a.cap);
          }
          if (mask) {
            int32_t token;
            uint32_t h;
            row_of(tid, token, h);
            const int32_t pos = before + token;
#pragma unroll
            for (int x = 0; x < kHalves; ++x)
#pragma unroll
              for (int v = 0; v < 16; ++v) {
                const int kk = 32 * (half + x) + 8 * (v / 4) + 4 * g + v % 4;
                const int32_t key = kb + kk;
                const bool off = (key >= k1) | ((a.causal != 0) & (key > pos)) | ((a.window >= 0) & (key < pos - a.window)) |
                                 ((bad >> (kk / 16) & 1) != 0);
                sc[x][v] = off ? -INFINITY : sc[x][v];
              }
          }
          const float scale = kCap != kNoCap ? 1.0f : a.scale_log2;
          float mx = sc[0][0];
#pragma unroll
          for (int x = 0; x < kHalves; ++x)
#pragma unroll
            for (int v = 0; v < 16; ++v) mx = fmaxf(mx, sc[x][v]);
          mx *= scale;
          if (__any(mx > top + kGrow)) {
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float now = mx > top ? mx : top;
            const float by = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - now);
            sum *= by;
#pragma unroll
            for (int d = 0; d < kDt; ++d)
#pragma unroll
              for (int v = 0; v < 16; ++v) o[d][v] *= by;
            top = now;
          }
          const float base = top == -INFINITY ? 0.0f : top;
          // Half after half: the exponentials of the second run beside the first's products.
#pragma unroll
          for (int x = 0; x < kHalves; ++x) {
            const auto value = [&](int n) {  // the operand of product n: 16 keys n / kDt, dims 32 (n % kDt) ..
              const uint32_t row = 16 * (2 * (half + x) + n / kDt) * 2 * D, d = n % kDt, swap = 64 * d | 16 * SwapOf<D>(0, d);
              const U2 lo = LdsTranspose(vt, (va[0] ^ swap) + row), hi = LdsTranspose(vt, (va[1] ^ swap) + row);
              return U4{lo[0], lo[1], hi[0], hi[1]};
            };
            U4 vv[kAhead];
            const auto ahead = [&] {
#pragma unroll
              for (int n = 0; n < kAhead; ++n) vv[n] = value(n);
            };
            if constexpr (D == 128) ahead();
            U4 p[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float y[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                y[e] = __builtin_amdgcn_exp2f(fmaf(sc[x][8 * c + e], scale, -base));
                sum += y[e];
              }
              p[c] = U4{PackBf16Rne(y[0], y[1]), PackBf16Rne(y[2], y[3]), PackBf16Rne(y[4], y[5]), PackBf16Rne(y[6], y[7])};
            }
            if constexpr (D == 128) {
              __builtin_amdgcn_sched_barrier(0);
            } else {
              ahead();
            }
#pragma unroll
            for (int n = 0; n < 2 * kDt; ++n) {
              const U4 v = vv[n % kAhead];
              if (n + kAhead < 2 * kDt) vv[n % kAhead] = value(n + kAhead);
              o[n % kDt] = Mfma32(v, p[n / kDt], o[n % kDt]);
            }
            // At 128 the first reads come in front of the exponentials and each product in front of the reads that it leaves room
            // for: 2% (two prompts of 3,500 to 4,096 tokens on prefixes, 32 heads over 8). At 64 and 256 that order is as fast or
            // faster.
            if constexpr (D == 128) {
#pragma unroll
              for (int n = 0; n < 2 * kDt; ++n) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
              }
              __builtin_amdgcn_sched_barrier(0);
            }
          }
          if (careful) {
            int32_t token;
            uint32_t h;
            row_of(tid, token, h);
            const int32_t pos = before + token;
            for (int kk = 32 * half; kk < 32 * (half + kHalves); ++kk) {
              const uint32_t blocks = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(lds.nan[slot][kk])));
              if (blocks == 0) continue;
              const int32_t key = kb + kk;
              if ((a.causal && key > pos) || (a.window >= 0 && key < pos - a.window)) continue;
#pragma unroll
              for (int d = 0; d < kDt; ++d) {
                if (blocks >> d & 1) {
#pragma unroll
                  for (int v = 0; v < 16; ++v) o[d][v] = NAN;
                }
              }
            }
          }
        }
      }
      if (t + 1 < tiles) store(t + 1, tid, careful);
    }
  };
  pass(false);
  bool nan = false;
#pragma unroll
  for (int d = 0; d < kDt; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) nan |= o[d][v] != o[d][v];
  if (__syncthreads_or(nan)) pass(true);

  sum += __shfl_xor(sum, 32);
  int32_t token;
  uint32_t h;
  row_of(tid, token, h);
  if (token < 0) return;
  const uint64_t at = static_cast<uint64_t>(s.first + token) * a.q_heads + h;
  if (range.parts > 1) {
    const uint64_t row = static_cast<uint64_t>(split) * a.tokens * a.q_heads + at;
#pragma unroll
    for (int d = 0; d < kDt; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        *reinterpret_cast<F4v*>(a.tile_o + row * D + 32 * d + 8 * i + 4 * g) =
            F4v{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
      }
    if (g == 0) a.tile_ml[2 * row] = top, a.tile_ml[2 * row + 1] = sum;
    return;
  }
  const float inv = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : NAN;
#pragma unroll
  for (int d = 0; d < kDt; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<U2*>(a.out + at * D + 32 * d + 8 * i + 4 * g) =
          U2{PackBf16Rne(o[d][4 * i] * inv, o[d][4 * i + 1] * inv), PackBf16Rne(o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv)};
    }
  if (a.lse != nullptr && g == 0) a.lse[at] = sum > 0.0f ? top + __builtin_amdgcn_logf(sum) : sum == sum ? -INFINITY : NAN;
}

// One row's parts by a workgroup: D / 4 lanes a part, their loads together, then the lanes' sums. The order of the additions is
// that of the parts' numbers, whichever workgroup wrote them when. row_of(p): part p's partial row; at: the output row.
template <int D, typename F>
__device__ __forceinline__ void MergeRow(const Args& a, const float* part_o, const float* part_ml, F&& row_of, uint32_t parts,
                                         uint64_t at) {
  constexpr uint32_t kLanes = D / 4, kGroups = 256 / kLanes, kAtOnce = 4;
  __shared__ float sums[kGroups][D + 4];
  __shared__ float totals[kGroups], tops[kGroups];
  const uint32_t group = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
  float top = -INFINITY, total = 0.0f;
  F4v y{0, 0, 0, 0};
  for (uint32_t p0 = group; p0 < parts; p0 += kGroups * kAtOnce) {
    float m[kAtOnce], l[kAtOnce];
    F4v v[kAtOnce];
#pragma unroll
    for (uint32_t i = 0; i < kAtOnce; ++i) {
      const uint32_t p = p0 + i * kGroups;
      m[i] = -INFINITY, l[i] = 0.0f, v[i] = F4v{0, 0, 0, 0};
      if (p < parts) {
        const uint64_t row = row_of(p);
        m[i] = part_ml[2 * row], l[i] = part_ml[2 * row + 1];
        v[i] = *reinterpret_cast<const F4v*>(part_o + row * D + d);
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < kAtOnce; ++i) {
      const float now = fmaxf(top, m[i]);
      const float old = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - now);
      const float by = m[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[i] - now);
      total = total * old + l[i] * by;
      y = y * old + v[i] * by;
      top = now;
    }
  }
  *reinterpret_cast<F4v*>(&sums[group][d]) = y;
  if (d == 0) totals[group] = total, tops[group] = top;
  __syncthreads();
  if (threadIdx.x >= kLanes) return;
  top = tops[0];
#pragma unroll
  for (uint32_t i = 1; i < kGroups; ++i) top = fmaxf(top, tops[i]);
  total = 0.0f, y = F4v{0, 0, 0, 0};
#pragma unroll
  for (uint32_t i = 0; i < kGroups; ++i) {
    const float by = tops[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(tops[i] - top);
    total += totals[i] * by;
    y += *reinterpret_cast<const F4v*>(&sums[i][d]) * by;
  }
  const float inv = total > 0.0f ? 1.0f / total : total == total ? 0.0f : NAN;
  *reinterpret_cast<U2*>(a.out + at * D + d) = U2{PackBf16Rne(y[0] * inv, y[1] * inv), PackBf16Rne(y[2] * inv, y[3] * inv)};
  if (a.lse != nullptr && d == 0) {
    a.lse[at] = total > 0.0f ? top + __builtin_amdgcn_logf(total) : total == total ? -INFINITY : NAN;
  }
}

// Block (tile and KV head, 1,024 / D rows of it): D / 4 lanes a row, up to four parts' loads together.
template <int D>
__global__ void __launch_bounds__(256) TileMergeKernel(Args a) {
  constexpr int32_t kLanes = D / 4, kRows = 256 / kLanes;
  const uint32_t head = blockIdx.x % a.cache.kv_heads;
  uint32_t b = 0;
  int32_t tile = 0;
  if (!FindTile(a, blockIdx.x / a.cache.kv_heads, 32 * kTileWaves, b, tile)) return;
  const Sequence s = SequenceOf(a, b);
  const TileKeys range = KeysOfTile(a, s, tile, 32 * kTileWaves);
  const int32_t group = static_cast<int32_t>(a.group);
  const int32_t row = tile * 32 * kTileWaves + static_cast<int32_t>(blockIdx.y * kRows + threadIdx.x / kLanes);
  if (range.parts <= 1 || row >= s.count * group) return;
  const int32_t token = row / group, d = static_cast<int32_t>(threadIdx.x) % kLanes * 4;
  const uint32_t h = head * a.group + static_cast<uint32_t>(row - token * group);
  const uint64_t at = static_cast<uint64_t>(s.first + token) * a.q_heads + h;
  const uint64_t step = static_cast<uint64_t>(a.tokens) * a.q_heads;
  float top = -INFINITY, total = 0.0f;
  F4v y{0, 0, 0, 0};
  for (uint32_t p0 = 0; p0 < range.parts; p0 += 4) {
    float m[4], l[4];
    F4v v[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      m[i] = -INFINITY, l[i] = 0.0f, v[i] = F4v{0, 0, 0, 0};
      if (p0 + i < range.parts) {
        const uint64_t r = (p0 + i) * step + at;
        m[i] = a.tile_ml[2 * r], l[i] = a.tile_ml[2 * r + 1];
        v[i] = *reinterpret_cast<const F4v*>(a.tile_o + r * D + d);
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const float now = fmaxf(top, m[i]);
      const float old = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - now);
      const float by = m[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[i] - now);
      total = total * old + l[i] * by;
      y = y * old + v[i] * by;
      top = now;
    }
  }
  const float inv = total > 0.0f ? 1.0f / total : total == total ? 0.0f : NAN;
  *reinterpret_cast<U2*>(a.out + at * D + d) = U2{PackBf16Rne(y[0] * inv, y[1] * inv), PackBf16Rne(y[2] * inv, y[3] * inv)};
  if (a.lse != nullptr && d == 0) {
    a.lse[at] = total > 0.0f ? top + __builtin_amdgcn_logf(total) : total == total ? -INFINITY : NAN;
  }
}

// A split sequence's parts. Block (row of a KV head, or the first of several, KV head, sequence).
template <int D>
__global__ void __launch_bounds__(256) RowMergeKernel(Args a) {
  const Sequence s = SequenceOf(a, blockIdx.z);
  const uint32_t all = a.cut[0], before = a.cut[1 + blockIdx.z], units = UnitsOf(a, s), heads = a.cache.kv_heads;
  if (units <= 1) return;
  const Deal deal(all * heads, a.places);
  const uint32_t begin = before * heads + blockIdx.y * units, first = deal.PlaceOf(begin), last = deal.PlaceOf(begin + units - 1);
  if (first == last) return;  // whole
  const int32_t group = static_cast<int32_t>(a.group);
  const uint64_t rows = static_cast<uint64_t>(a.short_tokens) * a.group;
  for (int32_t row = static_cast<int32_t>(blockIdx.x); row < s.count * group; row += static_cast<int32_t>(gridDim.x)) {
    const int32_t token = row / group;
    const uint32_t h = blockIdx.y * a.group + static_cast<uint32_t>(row - token * group);
    MergeRow<D>(a, a.part_o, a.part_ml,
                [&](uint32_t p) {
                  return (2 * static_cast<uint64_t>(first + p) + (p == 0 ? 1 : 0)) * rows + static_cast<uint32_t>(row);
                },
                last - first + 1, static_cast<uint64_t>(s.first + token) * a.q_heads + h);
    __syncthreads();
  }
}

// ---- Admission and launch --------------------------------------------------------------------------------------------------

// Into how many parts the tile kernel's keys are best cut, by what its workgroups were measured to take: 12 us (16 at head_dim
// 256) to begin and end, 1.25, 1.8 and 4.1 us for each 64 keys at head_dim 64, 128 and 256 on a CU of their own (at 64 a CU holds
// two, which then take twice as long), and for more parts than one the merge, 4 us, 0.97 for each part, and the partial rows once
// out and in at 8 TB/s (they stay in the last cache). With G tiles of all KV heads, G S / CUs rounds follow each other: whole ones
// where all tiles see as many keys, any number where a causal prompt's first tiles see few. Parts are whole 64 keys, so only an S
// that they come out at counts. Measured, us, without parts / with the S chosen here: 512 tokens behind 8,000, 32 heads over 8 of
// 128: 283 / 94 (4); 512 behind 500, 8 heads of 256 over 2: 80 / 38 (8); two of 100 behind 8,000, 32 heads over 8 of 64: 38 (8;
// 4 parts 56, 12 parts 44); 3,000 alone at 256: 211 / 93 (4); four of 1,000 to 2,000 on prefixes: 176 / 132 (2) at 256, and at 64,
// 32 heads over 8, 97 (2 parts: 124).
uint32_t TileSplits(const RoostAmdPagedAttentionF4Params& p, uint64_t groups, uint64_t keys, uint32_t cus) {
  const uint32_t d = p.cache.head_dim;
  const double ends = d == 256 ? 16 : 12, step = d == 256 ? 4.1 : d == 128 ? 1.8 : 1.25;
  const uint64_t steps = roost::CeilDiv(keys, kTileKeys);
  const double fresh = p.causal ? std::min<double>(p.max_q_len ? p.max_q_len : p.tokens, keys) : 0;
  const double mean = 1 - fresh / (2.0 * keys);  // of the keys that the last tile sees, what a tile does
  const double row_us = double(p.tokens) * p.q_heads * d * 8 / 8e6;
  uint32_t best = 1;
  double least = 0;
  for (uint32_t s = 1; s <= 16; ++s) {
    const uint64_t part = roost::CeilDiv(steps, s);
    if (roost::CeilDiv(steps, part) != s) continue;
    const double rounds = std::max(1.0, double(groups) * s / cus), one = ends + step * part;
    const double alike = std::ceil(rounds) * one, unlike = std::max(one, rounds * (ends + step * part * mean));
    const double us = (2 * mean - 1) * alike + (2 - 2 * mean) * unlike + (s > 1 ? 4 + s * (0.97 + row_us) : 0);
    if (s == 1 || us < least) best = s, least = us;
  }
  return best;
}

struct Cut {
  uint32_t row_tiles;     // of 16 rows in the row kernel
  uint32_t short_tokens;
  uint32_t places;        // its workgroups
  uint32_t merge_rows;    // of a KV head that its merge is expected to have
  bool merge;
  uint64_t rows;          // its partial rows
  bool by_row, by_tile;   // which kernels run
  uint32_t row_limit;
  uint32_t tiles, tile_splits;
  uint64_t tile_rows;     // its partial rows
};

Cut CutOf(const RoostAmdPagedAttentionF4Params& p, uint32_t cus) {
  Cut c{};
  const uint32_t group = p.q_heads / p.cache.kv_heads;
  const uint64_t most = p.kv_indptr.address != nullptr ? p.block_tables.length : p.max_blocks;
  uint64_t keys = p.max_kv_len ? p.max_kv_len : std::min<uint64_t>(most * p.cache.page_size, 16384);
  keys = std::min<uint64_t>(std::max<uint64_t>(keys, 1), kMostKeys);
  const auto seen = [&](uint64_t tokens) {
    return p.window_left < 0 ? keys : std::min<uint64_t>(keys, uint64_t{1} * p.window_left + 16 + tokens);
  };
  // Which kernels: sequences of up to 16 rows (32 where a token alone has more than 16) go row by row, longer ones by tiles. One
  // kernel is enough where no sequence is expected for the other; it then takes all, so an expectation that fails costs time only.
  // At head_dim 256 two tiles of 16 rows do not fit a wavefront's registers, and 32 rows take two turns.
  const uint64_t longest = p.max_q_len ? std::min(p.max_q_len, p.tokens) : p.tokens, expected = longest * group;
  c.row_tiles = p.cache.head_dim < 256 && (group > 16 || (expected > 16 && expected <= 32)) ? 2 : 1;
  const uint32_t few = std::max(16 * c.row_tiles, group);
  c.short_tokens = few / group;
  c.by_tile = expected > few;
  // A sequence has what the others leave of the tokens, at least. The row kernel's launches cost 8 us where it finds nothing.
  c.by_row = !c.by_tile || p.tokens <= (p.batch - 1) * longest + c.short_tokens;
  c.row_limit = !c.by_tile ? 0x7FFFFFFF : c.by_row ? few : 0;
  if (c.by_row) {
    // As many workgroups as the chip holds at once, or one for each unit of keys where fewer are expected; one for each KV head of
    // a batch that is too large to be dealt.
    const uint64_t least = uint64_t{p.batch} * p.cache.kv_heads, units = roost::CeilDiv(seen(c.short_tokens), kUnit);
    c.merge = p.batch <= kMaxScheduled;
    const uint64_t held = uint64_t{cus} * RowsResident(p.cache.head_dim, c.row_tiles);
    c.places = static_cast<uint32_t>(c.merge ? std::min(held, least * units) : least);
    c.merge_rows = std::min(c.short_tokens, p.max_q_len ? p.max_q_len : c.short_tokens) * group;
    c.rows = c.merge ? 2 * uint64_t{c.places} * c.short_tokens * group : 0;
  }
  c.tile_splits = 1;
  if (c.by_tile) {
    const uint64_t rows = 32 * kTileWaves, all = uint64_t{p.tokens} * group;
    const uint64_t longer = std::min<uint64_t>(p.batch, all / (c.row_limit + 1));  // sequences that it can have
    c.tiles = static_cast<uint32_t>(all / rows + longer);
    c.tile_splits = TileSplits(p, roost::CeilDiv(all, rows) * p.cache.kv_heads, seen(rows / group), cus);
    c.tile_rows = c.tile_splits > 1 ? uint64_t{c.tile_splits} * p.tokens * p.q_heads : 0;
  }
  return c;
}

uint64_t WorkspaceBytes(const RoostAmdPagedAttentionF4Params& p, const Cut& c) {
  return (c.rows + c.tile_rows) * (p.cache.head_dim + 2) * 4 + (c.merge ? 4 * (uint64_t{p.batch} + 1) : 0);
}

void AdmitLaunch(roost::Gate& gate, const RoostAmdPagedAttentionF4Params& p, const Cut& c) {
  gate.Expect(uint64_t{c.tiles} * p.cache.kv_heads * c.tile_splits < (1u << 23), ROOST_STATUS_UNSUPPORTED,
              "%u tokens of %u heads: more tiles than one launch takes", p.tokens, p.q_heads)
      .Expect(c.places < (1u << 24) - 8, ROOST_STATUS_UNSUPPORTED, "%u sequences of %u KV heads: more than one launch takes",
              p.batch, p.cache.kv_heads);
}

RoostStatus Admit(const RoostAmdPagedAttentionF4Params& p, uint64_t& pages) {
  roost::Gate gate(kOp);
  roost::AdmitCacheF4(gate, p.cache, pages);
  ROOST_GATE_RETURN(gate);
  const uint32_t d = p.cache.head_dim;
  gate.Expect(p.q_heads > 0 && p.q_heads % p.cache.kv_heads == 0 && p.q_heads / p.cache.kv_heads <= 32, ROOST_STATUS_UNSUPPORTED,
              "q_heads = %u over kv_heads = %u: 1 to 32 whole query heads to each are built", p.q_heads, p.cache.kv_heads)
      .Expect(p.tokens < (1u << 24) && p.batch <= 65535, ROOST_STATUS_UNSUPPORTED,
              "tokens = %u (below 2^24), batch = %u (at most 65,535)", p.tokens, p.batch)
      .Expect(uint64_t{p.tokens} * p.q_heads < (1u << 31), ROOST_STATUS_UNSUPPORTED, "%u tokens of %u heads: 2^31 rows or more",
              p.tokens, p.q_heads)
      .Expect(p.q.dtype == ROOST_DTYPE_BF16 && p.output.dtype == ROOST_DTYPE_BF16, ROOST_STATUS_UNSUPPORTED,
              "q is %s and output %s; both are bf16 here", roost::Describe(p.q.dtype).name, roost::Describe(p.output.dtype).name)
      .Expect(p.causal <= 1, ROOST_STATUS_INVALID_ARGUMENT, "causal = %u, not 0 or 1", p.causal)
      .Expect(p.window_left >= -1 && p.window_left <= kMostKeys, ROOST_STATUS_INVALID_ARGUMENT,
              "window_left = %d, not -1 to 2^30", p.window_left)
      .Expect(p.window_left < 0 || p.causal == 1, ROOST_STATUS_UNSUPPORTED, "a window without causal has no kernel here")
      .Expect(p.sm_scale >= 0.0f && p.sm_scale < INFINITY, ROOST_STATUS_INVALID_ARGUMENT,
              "sm_scale = %g is not 0 (1/sqrt(head_dim)) or positive and finite", p.sm_scale)
      .Expect(p.sm_scale <= 0x1p126f, ROOST_STATUS_UNSUPPORTED, "sm_scale = %g, above 2^126: its product with log2(e) passes f32",
              p.sm_scale)
      .Expect(p.logits_soft_cap >= 0.0f && p.logits_soft_cap < INFINITY, ROOST_STATUS_INVALID_ARGUMENT,
              "logits_soft_cap = %g is not 0 or positive and finite", p.logits_soft_cap);
  ROOST_GATE_RETURN(gate);
  if (p.tokens == 0 || p.batch == 0) return ROOST_STATUS_OK;
  const uint64_t width = uint64_t{p.q_heads} * d, stride = p.q_stride ? p.q_stride : width;
  const bool csr = p.kv_indptr.address != nullptr;
  gate.Expect(stride >= width && stride % 8 == 0, ROOST_STATUS_INVALID_ARGUMENT,
              "q_stride = %u: below a token's %llu or no multiple of 8", p.q_stride, static_cast<unsigned long long>(width))
      .Tensor("q", p.q, ROOST_DTYPE_BF16, (p.tokens - 1) * stride + width)
      .Tensor("output", p.output, ROOST_DTYPE_BF16, p.tokens * width)
      .OptionalTensor("lse", p.lse, ROOST_DTYPE_F32, uint64_t{p.tokens} * p.q_heads)
      .Tensor("cu_seqlens", p.cu_seqlens, ROOST_DTYPE_I32, p.batch + 1)
      .Expect(!csr || (p.max_blocks == 0 && p.table_rows == 0 && p.sequences.address == nullptr), ROOST_STATUS_INVALID_ARGUMENT,
              "kv_indptr goes without max_blocks, table_rows and sequences")
      .Expect(csr || (p.max_blocks > 0 && p.table_rows > 0), ROOST_STATUS_INVALID_ARGUMENT,
              "block_tables of %u x %u: empty", p.table_rows, p.max_blocks)
      .Expect(csr || p.sequences.address != nullptr || p.table_rows >= p.batch, ROOST_STATUS_INVALID_ARGUMENT,
              "%u table rows for a batch of %u without sequences", p.table_rows, p.batch);
  ROOST_GATE_RETURN(gate);
  gate.Tensor("block_tables", p.block_tables, ROOST_DTYPE_I32, csr ? 0 : uint64_t{p.table_rows} * p.max_blocks)
      .Expect(p.block_tables.address != nullptr || p.block_tables.length == 0, ROOST_STATUS_INVALID_ARGUMENT,
              "block_tables: address is NULL")
      .Tensor("kv_lens", p.kv_lens, ROOST_DTYPE_I32, csr ? p.batch : p.table_rows)
      .OptionalTensor("kv_indptr", p.kv_indptr, ROOST_DTYPE_I32, p.batch + 1)
      .OptionalTensor("sequences", p.sequences, ROOST_DTYPE_I32, p.batch)
      .Aligned("q", p.q.address, 16)
      .Aligned("output", p.output.address, 16)
      .Aligned("lse", p.lse.address, 4)
      .Aligned("cu_seqlens", p.cu_seqlens.address, 4)
      .Aligned("block_tables", p.block_tables.address, 4)
      .Aligned("kv_lens", p.kv_lens.address, 4)
      .Aligned("kv_indptr", p.kv_indptr.address, 4)
      .Aligned("sequences", p.sequences.address, 4);
  ROOST_GATE_RETURN(gate);
  const uint64_t page = uint64_t{p.cache.kv_heads} * p.cache.page_size * d / 32;
  const roost::Extent out = roost::ExtentOf(p.output.address, 2 * p.tokens * width);
  const roost::Extent lse = roost::ExtentOf(p.lse.address, 4 * uint64_t{p.tokens} * p.q_heads);
  for (const roost::Extent& other :
       {roost::ExtentOf(p.q.address, p.tokens, 2 * stride, 2 * width), roost::ExtentOf(p.cache.k.address, pages * page * 16),
        roost::ExtentOf(p.cache.v.address, pages * page * 16), roost::ExtentOf(p.cache.k_scales.address, pages * page),
        roost::ExtentOf(p.cache.v_scales.address, pages * page), roost::ExtentOf(p.cu_seqlens.address, 4 * (uint64_t{p.batch} + 1)),
        roost::ExtentOf(p.block_tables.address, 4 * p.block_tables.length),
        roost::ExtentOf(p.kv_lens.address, 4 * p.kv_lens.length), roost::ExtentOf(p.kv_indptr.address, 4 * (uint64_t{p.batch} + 1)),
        roost::ExtentOf(p.sequences.address, 4 * uint64_t{p.batch})}) {
    gate.Expect(!roost::Overlap(out, other) && !roost::Overlap(lse, other), ROOST_STATUS_INVALID_ARGUMENT,
                "output or lse overlaps an input of the call");
  }
  gate.Expect(!roost::Overlap(out, lse), ROOST_STATUS_INVALID_ARGUMENT, "output and lse overlap");
  return gate.status();
}

template <int D, int kCap>
void Launch(const Args& a, const Cut& c, hipStream_t s) {
  if (c.by_tile) TileAttentionKernel<D, kCap><<<c.tiles * a.cache.kv_heads * c.tile_splits, 64 * kTileWaves, 0, s>>>(a);
  if (c.by_tile && c.tile_splits > 1) {
    TileMergeKernel<D><<<dim3(c.tiles * a.cache.kv_heads, 32 * kTileWaves * D / 1024), 256, 0, s>>>(a);
  }
  if (!c.by_row) return;
  const uint32_t grid = (c.places + 7) / 8 * 8;  // whole rounds of the dies
  constexpr int kTiles = D == 256 ? 1 : 2;
  if (c.row_tiles < kTiles) {
    RowAttentionKernel<D, 1, kCap><<<grid, 64 * kRowWaves, 0, s>>>(a);
  } else {
    RowAttentionKernel<D, kTiles, kCap><<<grid, 64 * kRowWaves, 0, s>>>(a);
  }
  if (c.merge) {
    RowMergeKernel<D><<<dim3(c.merge_rows, a.cache.kv_heads, a.batch), 256, 0, s>>>(a);
  }
}

}  // namespace

extern "C" ROOST_API RoostStatus roost_amd_paged_attention_f4_workspace(RoostContext* ctx, const void* params,
                                                                        RoostWorkspaceSizes* sizes) {
  roost::Gate gate(kOp);
  gate.Expect(ctx != nullptr && sizes != nullptr, ROOST_STATUS_INVALID_ARGUMENT, "a context and a sizes record are required")
      .Header(params, sizeof(RoostAmdPagedAttentionF4Params));
  ROOST_GATE_RETURN(gate);
  gate.Header(sizes, sizeof(RoostWorkspaceSizes));
  ROOST_GATE_RETURN(gate);
  const auto& p = *static_cast<const RoostAmdPagedAttentionF4Params*>(params);
  return roost::CatchAll(kOp, [&]() -> RoostStatus {
    uint64_t pages = 0;
    ROOST_RETURN_IF_FAILED(Admit(p, pages));
    sizes->device_bytes = 0;
    if (p.tokens > 0 && p.batch > 0) {
      const Cut c = CutOf(p, ctx->compute_units);
      AdmitLaunch(gate, p, c);
      ROOST_GATE_RETURN(gate);
      sizes->device_bytes = WorkspaceBytes(p, c);
    }
    sizes->pinned_host_bytes = sizes->plan_bytes = 0;
    sizes->device_alignment = 256;
    return ROOST_STATUS_OK;
  });
}

extern "C" ROOST_API RoostStatus roost_amd_paged_attention_f4_run(RoostContext* ctx, const void* params,
                                                                  const RoostWorkspace* ws, void* stream) {
  roost::Gate gate(kOp);
  gate.Expect(ctx != nullptr, ROOST_STATUS_INVALID_ARGUMENT, "no context was passed")
      .Header(params, sizeof(RoostAmdPagedAttentionF4Params));
  ROOST_GATE_RETURN(gate);
  const auto& p = *static_cast<const RoostAmdPagedAttentionF4Params*>(params);
  return roost::CatchAll(kOp, [&]() -> RoostStatus {
    uint64_t pages = 0;
    ROOST_RETURN_IF_FAILED(Admit(p, pages));
    if (p.tokens == 0 || p.batch == 0) return ROOST_STATUS_OK;
    const Cut c = CutOf(p, ctx->compute_units);
    AdmitLaunch(gate, p, c);
    ROOST_GATE_RETURN(gate);
    const uint64_t bytes = WorkspaceBytes(p, c);
    gate.Expect(roost::HasDeviceRegion(ws, bytes), ROOST_STATUS_WORKSPACE_TOO_SMALL,
                "the call needs %llu bytes of 256-byte aligned device workspace", static_cast<unsigned long long>(bytes));
    ROOST_GATE_RETURN(gate);
    ROOST_GATE_RETURN(roost::OnDevice(gate, ctx));
    Args a{};
    a.q = static_cast<const uint16_t*>(p.q.address);
    a.out = static_cast<uint16_t*>(p.output.address);
    a.lse = static_cast<float*>(p.lse.address);
    a.cache = roost::ViewOf(p.cache, pages);
    a.cu = static_cast<const int32_t*>(p.cu_seqlens.address), a.tables = static_cast<const int32_t*>(p.block_tables.address);
    a.lens = static_cast<const int32_t*>(p.kv_lens.address), a.indptr = static_cast<const int32_t*>(p.kv_indptr.address);
    a.sequences = static_cast<const int32_t*>(p.sequences.address);
    a.q_stride = p.q_stride ? p.q_stride : uint64_t{p.q_heads} * p.cache.head_dim;
    a.table_entries = p.block_tables.length;
    a.batch = p.batch, a.tokens = p.tokens, a.q_heads = p.q_heads, a.group = p.q_heads / p.cache.kv_heads;
    a.table_rows = p.table_rows, a.max_blocks = p.max_blocks;
    const float scale = p.sm_scale != 0.0f ? p.sm_scale : 1.0f / std::sqrt(static_cast<float>(p.cache.head_dim));
    constexpr float kLog2e = 1.44269504f;
    a.scale_log2 = scale * kLog2e;
    const int kind = p.logits_soft_cap <= 0.0f ? kNoCap : p.logits_soft_cap <= kNearMost ? kNearCap : kFarCap;
    if (kind != kNoCap) {
      // Held to finite numbers at both ends: a cap times log2(e) may pass f32, and so may its reciprocal.
      const float cap = p.logits_soft_cap, capl = std::min(cap * kLog2e, FLT_MAX);
      a.cap = {capl, kind == kFarCap ? static_cast<float>(1 / (double{cap} * kLog2e)) : std::min(2.0f / cap, FLT_MAX)};
    }
    a.causal = p.causal, a.window = p.window_left;
    a.part_o = ws != nullptr ? static_cast<float*>(ws->device) : nullptr;
    a.part_ml = a.part_o + c.rows * p.cache.head_dim;
    a.tile_o = a.part_ml + 2 * c.rows;
    a.tile_ml = a.tile_o + c.tile_rows * p.cache.head_dim;
    a.cut = c.merge ? reinterpret_cast<uint32_t*>(a.tile_ml + 2 * c.tile_rows) : nullptr;
    a.places = c.places;
    a.max_units = std::min(65535u, 0xFFFFFFFFu / (kMaxScheduled * p.cache.kv_heads));
    a.short_tokens = c.short_tokens, a.row_limit = c.row_limit;
    a.tile_splits = c.tile_splits;
    const hipStream_t s = roost::Stream(stream);
    const auto launch = [&](auto cap) {
      constexpr int kCap = decltype(cap)::value;
      if (p.cache.head_dim == 64) {
        Launch<64, kCap>(a, c, s);
      } else if (p.cache.head_dim == 128) {
        Launch<128, kCap>(a, c, s);
      } else {
        Launch<256, kCap>(a, c, s);
      }
    };
    if (kind == kNoCap) {
      launch(std::integral_constant<int, kNoCap>{});
    } else if (kind == kNearCap) {
      launch(std::integral_constant<int, kNearCap>{});
    } else {
      launch(std::integral_constant<int, kFarCap>{});
    }
    return roost::HipStatus(hipGetLastError(), kOp, "kernel launch");
  });
}
