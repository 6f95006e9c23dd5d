// PagedAttentionF4 for gfx950: attention over a KV cache held in 4 bits, decode rows and prompt chunks.
//
// Per query row (a token's head) with KV head h: s_j = scale q . k_j over the keys j that the row sees, p = softmax(s),
// out = sum_j p_j v_j, in one pass over the keys with a running maximum and sum. K and V come as e2m1 codes with a power of two
// for each 32 dims, and become bf16 exactly (v_cvt_scalef32_pk_bf16_fp4, two codes an instruction, the scale included), so the
// products are those of the bf16 matrix instructions with f32 sums. Each p is rounded to bf16 once in front of its product.

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

struct SoftCap {  // cap tanh(s / cap) in log2 units: capl - 2 capl / (1 + 2^(k y)), y the scaled score
  float capl, k;
};
__device__ __forceinline__ float Capped(float y, SoftCap c) {
  return c.capl - 2.0f * c.capl * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y * c.k));
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
  uint32_t capped, causal;
  int32_t window;
  // How the work is cut.
  float *part_o, *part_ml;   // partial rows: sums before division, and (maximum, sum)
  uint32_t splits, part;     // a sequence's keys in at most `splits` parts of `part`, the last one open-ended
  uint32_t short_tokens;     // sequences of at most so many tokens may be split
  uint32_t row_limit;        // the row kernel takes sequences of at most so many rows, the tile kernel the others
  float *tile_o, *tile_ml;   // the tile kernel's partial rows, in at most tile_splits parts of its keys
  uint32_t tile_splits;
};

// ---- A sequence ---------------------------------------------------------------------------------------------------------

struct Sequence {
  int32_t first, count;   // tokens
  int32_t keys;
  int32_t blocks;         // entries at `pages`
  const int32_t* pages;
};

__device__ __forceinline__ Sequence SequenceOf(const Args& a, uint32_t b) {
  Sequence s;
  const int32_t most = static_cast<int32_t>(a.tokens);
  s.first = min(max(a.cu[b], 0), most);
  s.count = min(max(a.cu[b + 1], s.first), most) - s.first;
  const uint32_t shift = a.cache.page_shift;
  int64_t keys = 0;
  s.blocks = 0;
  s.pages = a.tables;
  if (a.indptr != nullptr) {
    const int64_t begin = a.indptr[b], end = min(static_cast<int64_t>(a.indptr[b + 1]), static_cast<int64_t>(a.table_entries));
    if (begin >= 0 && end > begin) {
      s.blocks = static_cast<int32_t>(end - begin);
      s.pages = a.tables + begin;
      keys = ((end - begin - 1) << shift) + min(max(a.lens[b], 0), 1 << shift);
    }
  } else {
    const int32_t row = a.sequences != nullptr ? a.sequences[b] : static_cast<int32_t>(b);
    if (static_cast<uint32_t>(row) < a.table_rows) {
      s.blocks = static_cast<int32_t>(a.max_blocks);
      s.pages = a.tables + static_cast<uint64_t>(row) * a.max_blocks;
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

// Parts that the keys [begin, end) of a sequence go in.
__device__ __forceinline__ uint32_t PartsOf(const Args& a, int32_t begin, int32_t end) {
  if (end <= begin) return 1;
  return min(static_cast<uint32_t>(end - begin + a.part - 1) / a.part, a.splits);
}

// ---- The row kernel -----------------------------------------------------------------------------------------------------------
// Up to 16 kTiles rows (a few tokens' query heads of one KV head) against one part of a sequence's keys: decode. Bound by the
// cache's bytes, 1.06 D a key and KV head.
//
// Operands of v_mfma_f32_16x16x32_bf16, lane l = 16 g + m: A[m][8 g + j], B[8 g + j][m], result [4 g + i][m].
//   S^T = K Q^T: key m of 16 as A, query row m as B. The contraction runs over the dims in any order, so lane (m, g) takes its
//   key's 16 bytes g, dims 32 g .. 32 g + 31 (head_dim 128): one scale a lane, word s the operand of step s, and 16 keys' codes
//   are one load of 1 KB.
//   O^T = V^T P^T: dim as A, keys contracted. Lane (m, g) of S^T holds rows' scores of keys 4 g + i of both 16-key groups; as B
//   it needs eight keys: those. So keys are contracted in the order 16 (j / 4) + 4 g + j % 4, and p goes from result to operand
//   without leaving the lane. A's lane (m, g) takes dims D / 16 m .. of those eight keys: one word a key (head_dim 128), eight
//   dims a lane, dim d of the word the operand of product d.
// Four wavefronts take the part's keys in turn by quarters; no barrier until their results meet in LDS.

constexpr int kRowWaves = 4;
constexpr int kStep = 32;  // keys a wavefront takes at a time

// Codes and scales of one step's keys in a lane.
template <int D>
struct RowStage {
  uint32_t k[2][D / 32];  // words of the lane's key in each group of 16
  uint32_t ks[2][D == 256 ? 2 : 1];
  uint32_t v[8][D == 256 ? 2 : 1];  // D = 64: the low half
  uint32_t vs[2];                   // four keys' scale bytes in each group
};

template <int D, int kTiles>
__global__ void __launch_bounds__(64 * kRowWaves) RowAttentionKernel(Args a) {
  constexpr int kWords = D / 32;   // of a lane's key
  constexpr int kDt = D / 16;      // dims of a lane's V word(s): products of 16 dims each
  constexpr int kBlocks = D / 32;
  __shared__ float red_o[kRowWaves][16][D];
  __shared__ float red_ml[kRowWaves][2][16];

  const uint32_t head = blockIdx.x, part = blockIdx.y;
  const Sequence s = SequenceOf(a, blockIdx.z);
  const int32_t rows = s.count * static_cast<int32_t>(a.group);
  if (rows == 0 || rows > static_cast<int32_t>(a.row_limit)) return;
  const int32_t begin = FirstKey(a, s, 0), end = s.keys;
  const bool split = s.count <= static_cast<int32_t>(a.short_tokens);
  const uint32_t parts = split ? PartsOf(a, begin, end) : 1;
  if (part >= parts) return;
  const int32_t k0 = begin + static_cast<int32_t>(part * a.part);
  const int32_t k1 = part + 1 == parts ? end : k0 + static_cast<int32_t>(a.part);

  const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // The wavefront's quarter, in whole steps.
  const int32_t steps = max(0, (k1 - k0 + kStep - 1) / kStep), each = (steps + kRowWaves - 1) / kRowWaves;
  const int32_t step0 = min(w * each, steps), my_steps = min(each, steps - step0);
  const int32_t my0 = k0 + step0 * kStep;
  const uint32_t shift = a.cache.page_shift, in_page = (1u << shift) - 1;

  // Page ids of 64 groups of 16 keys, one a lane; -1 for a page that is none.
  int32_t ids = -1;
  const auto load_ids = [&](int32_t step) {
    const int32_t key = my0 + step * kStep + 16 * lane, at = key >> shift;
    ids = -1;
    if (key < k1 && at < s.blocks) ids = s.pages[at];
    if (static_cast<uint32_t>(ids) >= a.cache.pages) ids = -1;
  };
  // A group's rows: its codes start at row * D / 2, its scales of block b at srow + (b << shift). Pages that are none: page 0,
  // whose keys are masked.
  const auto load = [&](int32_t step, RowStage<D>& st) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int32_t id = __builtin_amdgcn_readlane(ids, (2 * step + t) & 63);
      const uint32_t key = static_cast<uint32_t>(my0 + step * kStep + 16 * t) & in_page;
      const uint64_t head_page = static_cast<uint64_t>(max(id, 0)) * a.cache.kv_heads + head;
      const uint64_t row = (head_page << shift) + key;
      const uint64_t srow = ((head_page * kBlocks) << shift) + key;
      const uint8_t* kc = a.cache.k + row * (D / 2);
      const uint8_t* ksc = a.cache.k_scales + srow;
      const uint8_t* vc = a.cache.v + row * (D / 2);
      const uint8_t* vsc = a.cache.v_scales + srow;
      if constexpr (D == 64) {
        const U2 x = *reinterpret_cast<const U2*>(kc + m * 32 + 8 * g);
        st.k[t][0] = x[0], st.k[t][1] = x[1];
        st.ks[t][0] = ksc[((g >> 1) << shift) + m];
      } else {
#pragma unroll
        for (int h = 0; h < D / 128; ++h) {
          const U4 x = *reinterpret_cast<const U4*>(kc + m * (D / 2) + 64 * h + 16 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) st.k[t][4 * h + i] = x[i];
          st.ks[t][h] = ksc[((4 * h + g) << shift) + m];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* p = vc + (4 * g + i) * (D / 2) + m * (D / 32);
        if constexpr (D == 64) {
          st.v[4 * t + i][0] = *reinterpret_cast<const uint16_t*>(p);
        } else if constexpr (D == 128) {
          st.v[4 * t + i][0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
          const U2 x = *reinterpret_cast<const U2*>(p);
          st.v[4 * t + i][0] = x[0], st.v[4 * t + i][1] = x[1];
        }
      }
      st.vs[t] = *reinterpret_cast<const uint32_t*>(vsc + ((m / (512 / D)) << shift) + 4 * g);
    }
  };

  for (int32_t tile = 0; tile * 16 * kTiles < rows; ++tile) {
    // Query rows: lane m's of each 16.
    int32_t pos[kTiles];
    U4 q[kTiles][kWords];
    int64_t row_at[kTiles];  // token * q_heads + head, or -1
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      const int32_t r = (tile * kTiles + n) * 16 + m;
      const bool ok = r < rows;
      const int32_t token = ok ? r / static_cast<int32_t>(a.group) : 0;
      const uint32_t h = head * a.group + (ok ? r - token * static_cast<int32_t>(a.group) : 0);
      pos[n] = ok ? s.keys - s.count + token : -1;
      row_at[n] = ok ? static_cast<int64_t>(s.first + token) * a.q_heads + h : -1;
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
      const auto compute = [&](int32_t step, RowStage<D>& st) {
        const int32_t key0 = my0 + step * kStep;
        const int32_t id0 = __builtin_amdgcn_readlane(ids, (2 * step) & 63);
        const int32_t id1 = __builtin_amdgcn_readlane(ids, (2 * step + 1) & 63);
        const bool edge = key0 + kStep > k1 || (id0 | id1) < 0;
        const bool mask = edge || (a.causal && key0 + kStep > s.keys - s.count + 1) ||
                          (a.window >= 0 && key0 < s.keys - 1 - a.window);
        const auto absent = [&](int t, int i) {  // key 16 t + 4 g + i is none of the part's
          return key0 + 16 * t + 4 * g + i >= k1 || (t == 0 ? id0 : id1) < 0;
        };
        F4v sc[kTiles][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int n = 0; n < kTiles; ++n) sc[n][t] = F4v{0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            const float scale = F4Scale(st.ks[t][D == 256 ? i / 4 : 0]);
            const uint32_t c = st.k[t][i];
            const U4 kk{FromF4<0>(c, scale), FromF4<1>(c, scale), FromF4<2>(c, scale), FromF4<3>(c, scale)};
#pragma unroll
            for (int n = 0; n < kTiles; ++n) sc[n][t] = Mfma16(kk, q[n][i], sc[n][t]);
          }
        }
        float vscale[8];
        uint32_t nan_keys = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t byte = st.vs[t] >> (8 * i) & 0xFF;
            if (edge && absent(t, i)) byte = 127;  // whatever lies there: finite, times p = 0
            if (careful && byte > kF4ByteHigh) byte = 127, nan_keys |= 1u << (4 * t + i);
            vscale[4 * t + i] = F4Scale(byte);
          }
        }
        U4 p[kTiles];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          float y[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            y[j] = sc[n][j / 4][j % 4] * a.scale_log2;
            if (a.capped) y[j] = Capped(y[j], a.cap);
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
          float mx = y[0];
#pragma unroll
          for (int j = 1; j < 8; ++j) mx = fmaxf(mx, y[j]);
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
            y[j] = __builtin_amdgcn_exp2f(y[j] - base);
            sum[n] += y[j];
          }
          p[n] = U4{PackBf16Rne(y[0], y[1]), PackBf16Rne(y[2], y[3]), PackBf16Rne(y[4], y[5]), PackBf16Rne(y[6], y[7])};
        }
        // Two dims of eight keys, then each dim's eight keys.
        const auto two = [&](auto pair, int word, int out) {
          uint32_t c[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) c[j] = FromF4<decltype(pair)::value>(st.v[j][word], vscale[j]);
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
      };
      RowStage<D> even, odd;
      for (int32_t first = 0; first < my_steps; first += 32) {  // 64 groups' page ids
        load_ids(first);
        const int32_t last = min(my_steps, first + 32);
        load(first, even);
        for (int32_t i = first; i < last; i += 2) {
          if (i + 1 < last) load(i + 1, odd);
          compute(i, even);
          if (i + 1 >= last) break;
          if (i + 2 < last) load(i + 2, even);
          compute(i + 1, odd);
        }
      }
    };
    pass(false);
    bool nan = false;
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int d = 0; d < kDt; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) nan |= o[n][d][i] != o[n][d][i];
    if (__any(nan)) pass(true);

    // The four wavefronts' results meet, 16 rows at a time.
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      float l = sum[n];
      l += __shfl_xor(l, 16);
      l += __shfl_xor(l, 32);
      if (n > 0 || tile > 0) __syncthreads();  // the rows before are read
      if (g == 0) red_ml[w][0][m] = top[n], red_ml[w][1][m] = l;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < kDt; d += 4) {
          *reinterpret_cast<F4v*>(&red_o[w][m][(4 * g + i) * kDt + d]) =
              F4v{o[n][d][i], o[n][d + 1][i], o[n][d + 2][i], o[n][d + 3][i]};
        }
      __syncthreads();
      constexpr int kThreadsPerRow = 16, kPer = D / kThreadsPerRow;  // 16 rows x 16 threads
      const int r = threadIdx.x / kThreadsPerRow, d0 = (threadIdx.x % kThreadsPerRow) * kPer;
      const int32_t row = (tile * kTiles + n) * 16 + r;
      if (row >= rows) continue;
      float big = red_ml[0][0][r];
#pragma unroll
      for (int x = 1; x < kRowWaves; ++x) big = fmaxf(big, red_ml[x][0][r]);
      float total = 0.0f, f[kRowWaves], y[kPer];
#pragma unroll
      for (int x = 0; x < kRowWaves; ++x) {
        f[x] = red_ml[x][0][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(red_ml[x][0][r] - big);
        total += red_ml[x][1][r] * f[x];
      }
#pragma unroll
      for (int d = 0; d < kPer; ++d) {
        y[d] = 0.0f;
#pragma unroll
        for (int x = 0; x < kRowWaves; ++x) y[d] += red_o[x][r][d0 + d] * f[x];
      }
      const int32_t token = row / static_cast<int32_t>(a.group);
      const uint32_t h = head * a.group + static_cast<uint32_t>(row - token * static_cast<int32_t>(a.group));
      if (parts > 1) {
        const uint64_t at = ((static_cast<uint64_t>(blockIdx.z) * a.splits + part) * a.short_tokens + token) * a.q_heads + h;
#pragma unroll
        for (int d = 0; d < kPer; d += 4) {
          *reinterpret_cast<F4v*>(a.part_o + at * D + d0 + d) = F4v{y[d], y[d + 1], y[d + 2], y[d + 3]};
        }
        if (d0 == 0) a.part_ml[2 * at] = big, a.part_ml[2 * at + 1] = total;
        continue;
      }
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
}

// ---- The tile kernel ----------------------------------------------------------------------------------------------------------
// 32 kWaves rows of one sequence and KV head (rows are its tokens' query heads, token by token) against the keys that they see, 64
// at a time: prompt chunks. Bound by the matrix instructions and, beside them, by LDS reads and the softmax.
//
// A tile's codes come through registers, a lane a block of 32 dims (16 bytes, one scale), and go to LDS as bf16 once for all
// wavefronts: 64 conversions a lane and tile at head_dim 128 and 256 rows, where converting in each wavefront would take 192. Codes
// of the next tile are under way during a tile's products; LDS holds two tiles, so there is one barrier a tile.
//
// v_mfma_f32_32x32x16_bf16, lane l = 32 g + m: A[m][8 g + j], B[8 g + j][m], result register v at [8 (v / 4) + 4 g + v % 4][m].
//   S^T = K Q^T with 32 keys as A and the wavefront's 32 rows as B. A lane then holds, of its row, keys 4 g + i of each 8; the
//   products O^T = V^T P^T contract the keys in that order, so p stays in its lane, and V^T's operand (dim m, four keys twice) is
//   read from LDS by transposing reads.
// LDS: K rows are padded by 16 bytes, so that 16 keys' reads of 16 bytes meet no bank twice; V's 64-byte chunks are swizzled by
// the key, and their 16-byte pieces by the next bits of it, which does the same for the transposing reads of 8 keys x 64 bytes.

constexpr int kTileKeys = 64;

typedef __attribute__((address_space(3))) unsigned char LdsByte;

__device__ __forceinline__ U2 LdsTranspose(const unsigned char* base, uint32_t off) {
  auto* p = reinterpret_cast<__attribute__((address_space(3))) I4h*>(const_cast<LdsByte*>((const LdsByte*)base + off));
  return __builtin_bit_cast(U2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
}

template <int D>
struct TileLds {
  static constexpr int kKeyRow = 2 * D + 16;
  unsigned char k[2][kTileKeys * kKeyRow];
  unsigned char v[2][kTileKeys * 2 * D];
  uint32_t bad[3];                // groups of 16 keys without a page, of this tile, the next and the one after
  uint32_t nan[3][kTileKeys];     // blocks of V that are NaN; only kept in a careful pass
};

// Where block `block`, piece `piece` (8 dims) of a key lies in LDS.
template <int D>
__device__ __forceinline__ uint32_t ValueAt(uint32_t key, uint32_t block, uint32_t piece) {
  const uint32_t swap = D == 64 ? key >> 1 & 1 : key & 3;
  return key * 2 * D + ((block ^ swap) * 64) + ((piece ^ (key >> 2 & 3)) * 16);
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
    uint32_t end = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = static_cast<uint32_t>(__shfl_up(static_cast<int>(end), d));
      if (lane >= d) end += o;
    }
    const uint64_t here = __ballot(rank < end);
    if (here != 0) {
      const int at = __builtin_ctzll(here);
      b = base + static_cast<uint32_t>(at);
      tile = static_cast<int32_t>(__builtin_amdgcn_readlane(static_cast<int>(end), at)) - 1 - static_cast<int32_t>(rank);
      return true;
    }
    rank -= static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(end), 63));
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

template <int D, int kWaves, bool kCap>
__global__ void __launch_bounds__(64 * kWaves, kWaves / 4) TileAttentionKernel(Args a) {
  constexpr int kThreads = 64 * kWaves, kRows = 32 * kWaves;
  constexpr int kKs = D / 16, kDt = D / 32;
  constexpr int kPieces = (4 * D + kThreads - 1) / kThreads;  // blocks of 32 codes that a lane stages
  __shared__ __attribute__((aligned(16))) TileLds<D> lds;

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
  const int32_t tiles = k1 > k0 ? (k1 - k0 + kTileKeys - 1) / kTileKeys : 0;

  const int tid = threadIdx.x, lane = tid & 63, m = lane & 31, g = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t group = static_cast<int32_t>(a.group), rows = s.count * group;
  const int32_t r = tile * kRows + 32 * w + m;
  const bool row_ok = r < rows;
  const int32_t token = row_ok ? r / group : 0;
  const uint32_t h = head * a.group + static_cast<uint32_t>(row_ok ? r - token * group : 0);
  const int32_t before = s.keys - s.count;  // the first token's position
  const int32_t pos = before + token;
  // Positions of the wavefront's first and last row.
  const int32_t low = before + (tile * kRows + 32 * w) / group;
  const int32_t high = before + min((tile * kRows + 32 * w + 31) / group, s.count - 1);
  const bool idle = tile * kRows + 32 * w >= rows;  // the wavefront has no row, and only stages
  const uint64_t at = static_cast<uint64_t>(s.first + token) * a.q_heads + h;

  U4 q[kKs];
  {
    const uint16_t* qr = a.q + static_cast<uint64_t>(s.first + token) * a.q_stride + static_cast<uint64_t>(h) * D + 8 * g;
#pragma unroll
    for (int i = 0; i < kKs; ++i) {
      const U4 x = *reinterpret_cast<const U4*>(qr + 16 * i);
      q[i] = row_ok ? x : U4{0, 0, 0, 0};
    }
  }

  // Staging: piece tid + i kThreads of [K, V] x 64 keys x blocks.
  const uint32_t shift = a.cache.page_shift, in_page = (1u << shift) - 1;
  const auto piece_of = [&](int i, bool& value, int32_t& key, uint32_t& block) {
    const int p = tid + i * kThreads;
    value = p >= 2 * D;
    key = (p & (2 * D - 1)) / (D / 32);
    block = static_cast<uint32_t>(p) & (D / 32 - 1);
    return p < 4 * D;
  };
  int32_t ids[kPieces];
  U4 codes[kPieces];
  uint32_t scales[kPieces];
  const auto load_ids = [&](int32_t t) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      bool value;
      int32_t key;
      uint32_t block;
      ids[i] = -1;
      if (!piece_of(i, value, key, block) || t >= tiles) continue;
      const int32_t k = k0 + t * kTileKeys + key, entry = k >> shift;
      if ((k & ~15) < k1 && entry < s.blocks) ids[i] = s.pages[entry];
    }
  };
  const auto load_codes = [&](int32_t t) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      bool value;
      int32_t key;
      uint32_t block;
      if (!piece_of(i, value, key, block)) continue;
      if (static_cast<uint32_t>(ids[i]) >= a.cache.pages) ids[i] = -1;
      const uint32_t within = static_cast<uint32_t>(k0 + t * kTileKeys + key) & in_page;
      const uint64_t head_page = static_cast<uint64_t>(max(ids[i], 0)) * a.cache.kv_heads + head;
      codes[i] = *reinterpret_cast<const U4*>((value ? a.cache.v : a.cache.k) + ((head_page << shift) + within) * (D / 2) + 16 * block);
      scales[i] = (value ? a.cache.v_scales : a.cache.k_scales)[((head_page * (D / 32) + block) << shift) + within];
      if (ids[i] < 0) scales[i] |= 0x100;  // no key
    }
  };
  const auto store = [&](int32_t t, bool careful) {
    const int slot = t % 3;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      bool value;
      int32_t key;
      uint32_t block;
      if (!piece_of(i, value, key, block)) continue;
      const bool none = (scales[i] & 0x100) != 0;
      if (none && block == 0) atomicOr(&lds.bad[slot], 1u << (key / 16));
      uint32_t byte = scales[i] & 0xFF;
      if (value) {
        if (none || k0 + t * kTileKeys + key >= k1) byte = 127;  // whatever lies there: finite, times p = 0
        if (careful && byte > kF4ByteHigh) {
          byte = 127;
          atomicOr(&lds.nan[slot][key], 1u << block);
        }
      }
      const float scale = F4Scale(byte);
      unsigned char* const to = value ? lds.v[t & 1] : lds.k[t & 1];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t c = codes[i][j];
        const U4 x{FromF4<0>(c, scale), FromF4<1>(c, scale), FromF4<2>(c, scale), FromF4<3>(c, scale)};
        const uint32_t off = value ? ValueAt<D>(key, block, j) : key * TileLds<D>::kKeyRow + 64 * block + 16 * j;
        *reinterpret_cast<U4*>(to + off) = x;
      }
    }
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
    if (careful && tid < 64) lds.nan[0][tid] = lds.nan[1][tid] = lds.nan[2][tid] = 0;
    __syncthreads();
    if (tiles > 0) {
      load_ids(0);
      load_codes(0);
      load_ids(1);
      store(0, careful);
    }
    for (int32_t t = 0; t < tiles; ++t) {
      __syncthreads();  // tile t is in LDS; nobody reads tile t - 1 any more
      const int slot = t % 3, after = (t + 2) % 3;
      if (tid == 0) lds.bad[after] = 0;
      if (careful && tid < 64) lds.nan[after][tid] = 0;
      if (t + 1 < tiles) {
        load_codes(t + 1);
        load_ids(t + 2);
      }
      const int32_t kb = k0 + t * kTileKeys;
      if (!idle && !(a.causal && kb > high)) {
        const uint32_t bad = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(lds.bad[slot])));
        const bool mask = kb + kTileKeys > k1 || (a.causal && kb + kTileKeys - 1 > low) || bad != 0 ||
                          (a.window >= 0 && kb < high - a.window);
        const unsigned char* kt = lds.k[t & 1] + m * TileLds<D>::kKeyRow + 16 * g;
        const unsigned char* vt = lds.v[t & 1];
        // The transposing read of four keys x 16 dims by 16 lanes: lane 16 c + j addresses key j / 4, dims 4 (j % 4) of it.
        const uint32_t j = lane & 15, key4 = 4 * g + j / 4, piece = 2 * (lane >> 4 & 1) + (j % 4) / 2;
        uint32_t va[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) va[f] = ValueAt<D>(key4 + 8 * f, 0, piece) + 8 * (j & 1);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (a.causal && kb + 32 * half > high) break;
          F16v sc;
#pragma unroll
          for (int v = 0; v < 16; ++v) sc[v] = 0.0f;
#pragma unroll
          for (int i = 0; i < kKs; ++i) {
            sc = Mfma32(*reinterpret_cast<const U4*>(kt + 32 * half * TileLds<D>::kKeyRow + 32 * i), q[i], sc);
          }
          if constexpr (kCap) {
#pragma unroll
            for (int v = 0; v < 16; ++v) sc[v] = Capped(sc[v] * a.scale_log2, a.cap);
          }
          if (mask) {
#pragma unroll
            for (int v = 0; v < 16; ++v) {
              const int kk = 32 * half + 8 * (v / 4) + 4 * g + v % 4;
              const int32_t key = kb + kk;
              const bool off = (key >= k1) | ((a.causal != 0) & (key > pos)) | ((a.window >= 0) & (key < pos - a.window)) |
                               ((bad >> (kk / 16) & 1) != 0);
              sc[v] = off ? -INFINITY : sc[v];
            }
          }
          const float scale = kCap ? 1.0f : a.scale_log2;
          float mx = sc[0];
#pragma unroll
          for (int v = 1; v < 16; ++v) mx = fmaxf(mx, sc[v]);
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
          U4 p[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              y[e] = __builtin_amdgcn_exp2f(fmaf(sc[8 * c + e], scale, -base));
              sum += y[e];
            }
            p[c] = U4{PackBf16Rne(y[0], y[1]), PackBf16Rne(y[2], y[3]), PackBf16Rne(y[4], y[5]), PackBf16Rne(y[6], y[7])};
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int d = 0; d < kDt; ++d) {
              const uint32_t row = 16 * (2 * half + c) * 2 * D;
              const U2 lo = LdsTranspose(vt, (va[0] ^ (64 * d)) + row), hi = LdsTranspose(vt, (va[1] ^ (64 * d)) + row);
              o[d] = Mfma32(U4{lo[0], lo[1], hi[0], hi[1]}, p[c], o[d]);
            }
          }
          if (careful) {
            for (int kk = 32 * half; kk < 32 * half + 32; ++kk) {
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
      if (t + 1 < tiles) store(t + 1, careful);
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
  if (!row_ok) return;
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

// One row's parts, in order, by a wavefront. first: its first partial row, `step` rows between parts; at: its output row.
template <int D>
__device__ __forceinline__ void MergeRow(const Args& a, const float* part_o, const float* part_ml, uint64_t first, uint64_t step,
                                         uint32_t parts, uint64_t at) {
  constexpr int kPer = D / 64;
  const int lane = threadIdx.x & 63;
  float big = -INFINITY;
  for (uint32_t p = lane; p < parts; p += 64) big = fmaxf(big, part_ml[2 * (first + p * step)]);
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) big = fmaxf(big, __shfl_xor(big, x));
  float total = 0.0f, y[kPer] = {};
  for (uint32_t p = 0; p < parts; ++p) {
    const uint64_t row = first + p * step;
    const float m = part_ml[2 * row];
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - big);
    total += part_ml[2 * row + 1] * f;
#pragma unroll
    for (int d = 0; d < kPer; ++d) y[d] += part_o[row * D + lane * kPer + d] * f;
  }
  const float inv = total > 0.0f ? 1.0f / total : total == total ? 0.0f : NAN;
#pragma unroll
  for (int d = 0; d < kPer; ++d) a.out[at * D + lane * kPer + d] = static_cast<uint16_t>(PackBf16Rne(y[d] * inv, 0.0f));
  if (a.lse != nullptr && lane == 0) {
    a.lse[at] = total > 0.0f ? big + __builtin_amdgcn_logf(total) : total == total ? -INFINITY : NAN;
  }
}

// Block (tile and KV head, rows by fours).
template <int D, int kWaves>
__global__ void __launch_bounds__(256) TileMergeKernel(Args a) {
  const uint32_t head = blockIdx.x % a.cache.kv_heads;
  uint32_t b = 0;
  int32_t tile = 0;
  if (!FindTile(a, blockIdx.x / a.cache.kv_heads, 32 * kWaves, b, tile)) return;
  const Sequence s = SequenceOf(a, b);
  const TileKeys range = KeysOfTile(a, s, tile, 32 * kWaves);
  const int32_t group = static_cast<int32_t>(a.group);
  const int32_t row = tile * 32 * kWaves + static_cast<int32_t>(blockIdx.y * 4 + threadIdx.x / 64);
  if (range.parts <= 1 || row >= s.count * group) return;
  const int32_t token = row / group;
  const uint64_t at = static_cast<uint64_t>(s.first + token) * a.q_heads + head * a.group + static_cast<uint32_t>(row - token * group);
  MergeRow<D>(a, a.tile_o, a.tile_ml, at, static_cast<uint64_t>(a.tokens) * a.q_heads, range.parts, at);
}

// A split sequence's parts. Block (rows of a KV head by fours, KV head, sequence).
template <int D>
__global__ void __launch_bounds__(256) RowMergeKernel(Args a) {
  const Sequence s = SequenceOf(a, blockIdx.z);
  const int32_t group = static_cast<int32_t>(a.group), rows = s.count * group;
  const int32_t row = static_cast<int32_t>(blockIdx.x * 4 + threadIdx.x / 64);
  if (row >= rows || rows > static_cast<int32_t>(a.row_limit) || s.count > static_cast<int32_t>(a.short_tokens)) return;
  const uint32_t parts = PartsOf(a, FirstKey(a, s, 0), s.keys);
  if (parts <= 1) return;
  const int32_t token = row / group;
  const uint32_t h = blockIdx.y * a.group + static_cast<uint32_t>(row - token * group);
  const uint64_t step = static_cast<uint64_t>(a.short_tokens) * a.q_heads;
  const uint64_t first = static_cast<uint64_t>(blockIdx.z) * a.splits * step + static_cast<uint64_t>(token) * a.q_heads + h;
  MergeRow<D>(a, a.part_o, a.part_ml, first, step, parts, static_cast<uint64_t>(s.first + token) * a.q_heads + h);
}

// ---- Admission and launch --------------------------------------------------------------------------------------------------

constexpr int TileWaves(uint32_t d) { return d == 256 ? 4 : 8; }

struct Cut {
  uint32_t row_tiles;     // of 16 rows in the row kernel
  uint32_t splits, part, short_tokens;
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
  const uint64_t expected = uint64_t{p.max_q_len ? std::min(p.max_q_len, p.tokens) : p.tokens} * group;
  c.row_tiles = group > 16 || (expected > 16 && expected <= 32) ? 2 : 1;
  const uint32_t few = 16 * c.row_tiles;
  c.short_tokens = few / group;
  c.by_tile = expected > few;
  c.by_row = !c.by_tile || p.batch > 1;
  c.row_limit = !c.by_tile ? 0x7FFFFFFF : c.by_row ? few : 0;
  if (c.by_row) {
    const uint64_t wanted = roost::CeilDiv(4 * cus, std::max<uint64_t>(1, uint64_t{p.batch} * p.cache.kv_heads));
    const uint64_t k = seen(c.short_tokens), splits = std::max<uint64_t>(1, std::min<uint64_t>(wanted, roost::CeilDiv(k, 128)));
    c.part = static_cast<uint32_t>(roost::RoundUp(roost::CeilDiv(k, splits), 64));
    c.splits = static_cast<uint32_t>(roost::CeilDiv(k, c.part));
    c.rows = c.splits > 1 ? uint64_t{p.batch} * c.splits * c.short_tokens * p.q_heads : 0;
  } else {
    c.splits = 1, c.part = kMostKeys;
  }
  c.tile_splits = 1;
  if (c.by_tile) {
    const uint64_t rows = 32 * TileWaves(p.cache.head_dim), all = uint64_t{p.tokens} * group;
    const uint64_t longer = std::min<uint64_t>(p.batch, all / (c.row_limit + 1));  // sequences that it can have
    c.tiles = static_cast<uint32_t>(all / rows + longer);
    const uint64_t groups = std::max<uint64_t>(1, roost::CeilDiv(all, rows) * p.cache.kv_heads);
    if (4 * groups < 3 * cus) c.tile_splits = static_cast<uint32_t>(std::max<uint64_t>(1, std::min(cus / groups, seen(p.tokens) / 512)));
    c.tile_rows = c.tile_splits > 1 ? uint64_t{c.tile_splits} * p.tokens * p.q_heads : 0;
  }
  return c;
}

uint64_t WorkspaceBytes(const RoostAmdPagedAttentionF4Params& p, uint32_t cus) {
  const Cut c = CutOf(p, cus);
  return (c.rows + c.tile_rows) * (p.cache.head_dim + 2) * 4;
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
        roost::ExtentOf(p.block_tables.address, 4 * p.block_tables.length), roost::ExtentOf(p.kv_lens.address, 4 * p.kv_lens.length),
        roost::ExtentOf(p.kv_indptr.address, 4 * (uint64_t{p.batch} + 1)),
        roost::ExtentOf(p.sequences.address, 4 * uint64_t{p.batch})}) {
    gate.Expect(!roost::Overlap(out, other) && !roost::Overlap(lse, other), ROOST_STATUS_INVALID_ARGUMENT,
                "output or lse overlaps an input of the call");
  }
  gate.Expect(!roost::Overlap(out, lse), ROOST_STATUS_INVALID_ARGUMENT, "output and lse overlap");
  return gate.status();
}

template <int D, int kWaves>
void LaunchTiles(const Args& a, const Cut& c, hipStream_t s) {
  const uint32_t grid = c.tiles * a.cache.kv_heads * c.tile_splits;
  if (a.capped) {
    TileAttentionKernel<D, kWaves, true><<<grid, 64 * kWaves, 0, s>>>(a);
  } else {
    TileAttentionKernel<D, kWaves, false><<<grid, 64 * kWaves, 0, s>>>(a);
  }
  if (c.tile_splits > 1) TileMergeKernel<D, kWaves><<<dim3(c.tiles * a.cache.kv_heads, 8 * kWaves), 256, 0, s>>>(a);
}

template <int D>
void Launch(const Args& a, const Cut& c, hipStream_t s) {
  if (c.by_tile) LaunchTiles<D, TileWaves(D)>(a, c, s);
  if (!c.by_row) return;
  const dim3 grid(a.cache.kv_heads, c.splits, a.batch);
  if (c.row_tiles == 1) {
    RowAttentionKernel<D, 1><<<grid, 64 * kRowWaves, 0, s>>>(a);
  } else {
    RowAttentionKernel<D, 2><<<grid, 64 * kRowWaves, 0, s>>>(a);
  }
  if (c.splits > 1) {
    RowMergeKernel<D><<<dim3((c.short_tokens * a.group + 3) / 4, a.cache.kv_heads, a.batch), 256, 0, s>>>(a);
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
    sizes->device_bytes = WorkspaceBytes(p, ctx->compute_units);
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
    const uint64_t bytes = WorkspaceBytes(p, ctx->compute_units);
    gate.Expect(roost::HasDeviceRegion(ws, bytes), ROOST_STATUS_WORKSPACE_TOO_SMALL,
                "the call needs %llu bytes of 256-byte aligned device workspace", static_cast<unsigned long long>(bytes));
    ROOST_GATE_RETURN(gate);
    if (p.tokens == 0 || p.batch == 0) return ROOST_STATUS_OK;
    ROOST_GATE_RETURN(roost::OnDevice(gate, ctx));
    const Cut c = CutOf(p, ctx->compute_units);
    gate.Expect(uint64_t{c.tiles} * p.cache.kv_heads * c.tile_splits < (1u << 23), ROOST_STATUS_UNSUPPORTED,
                "%u tokens of %u heads: more tiles than one launch takes", p.tokens, p.q_heads);
    ROOST_GATE_RETURN(gate);
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
    a.capped = p.logits_soft_cap > 0.0f;
    if (a.capped) a.cap = {p.logits_soft_cap * kLog2e, 2.0f / p.logits_soft_cap};
    a.causal = p.causal, a.window = p.window_left;
    a.part_o = ws != nullptr ? static_cast<float*>(ws->device) : nullptr;
    a.part_ml = a.part_o + c.rows * p.cache.head_dim;
    a.tile_o = a.part_ml + 2 * c.rows;
    a.tile_ml = a.tile_o + c.tile_rows * p.cache.head_dim;
    a.splits = c.splits, a.part = c.part, a.short_tokens = c.short_tokens, a.row_limit = c.row_limit;
    a.tile_splits = c.tile_splits;
    const hipStream_t s = roost::Stream(stream);
    if (p.cache.head_dim == 64) {
      Launch<64>(a, c, s);
    } else if (p.cache.head_dim == 128) {
      Launch<128>(a, c, s);
    } else {
      Launch<256>(a, c, s);
    }
    return roost::HipStatus(hipGetLastError(), kOp, "kernel launch");
  });
}
