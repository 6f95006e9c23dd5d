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
typedef __bf16 B8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ F4v Mfma16(U4 a, U4 b, F4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(B8, a), __builtin_bit_cast(B8, b), c, 0, 0, 0);
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

// A split sequence's parts, in order. Block (rows of a KV head by fours, KV head, sequence), a wavefront a row.
template <int D>
__global__ void __launch_bounds__(256) RowMergeKernel(Args a) {
  const Sequence s = SequenceOf(a, blockIdx.z);
  const int32_t rows = s.count * static_cast<int32_t>(a.group);
  const int32_t row = static_cast<int32_t>(blockIdx.x * 4 + threadIdx.x / 64);
  if (row >= rows || rows > static_cast<int32_t>(a.row_limit) || s.count > static_cast<int32_t>(a.short_tokens)) return;
  const uint32_t parts = PartsOf(a, FirstKey(a, s, 0), s.keys);
  if (parts <= 1) return;
  const int lane = threadIdx.x & 63;
  constexpr int kPer = D / 64;
  const int32_t token = row / static_cast<int32_t>(a.group);
  const uint32_t h = blockIdx.y * a.group + static_cast<uint32_t>(row - token * static_cast<int32_t>(a.group));
  const uint64_t step = static_cast<uint64_t>(a.short_tokens) * a.q_heads;
  const uint64_t first = static_cast<uint64_t>(blockIdx.z) * a.splits * step + static_cast<uint64_t>(token) * a.q_heads + h;
  float big = -INFINITY;
  for (uint32_t p = lane; p < parts; p += 64) big = fmaxf(big, a.part_ml[2 * (first + p * step)]);
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) big = fmaxf(big, __shfl_xor(big, x));
  float total = 0.0f, y[kPer] = {};
  for (uint32_t p = 0; p < parts; ++p) {
    const uint64_t at = first + p * step;
    const float m = a.part_ml[2 * at];
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - big);
    total += a.part_ml[2 * at + 1] * f;
#pragma unroll
    for (int d = 0; d < kPer; ++d) y[d] += a.part_o[at * D + lane * kPer + d] * f;
  }
  const float inv = total > 0.0f ? 1.0f / total : total == total ? 0.0f : NAN;
  const uint64_t at = static_cast<uint64_t>(s.first + token) * a.q_heads + h;
#pragma unroll
  for (int d = 0; d < kPer; ++d) a.out[at * D + lane * kPer + d] = static_cast<uint16_t>(PackBf16Rne(y[d] * inv, 0.0f));
  if (a.lse != nullptr && lane == 0) {
    a.lse[at] = total > 0.0f ? big + __builtin_amdgcn_logf(total) : total == total ? -INFINITY : NAN;
  }
}

// ---- Admission and launch --------------------------------------------------------------------------------------------------

struct Cut {
  uint32_t tiles;         // of 16 rows in the row kernel
  uint32_t splits, part, short_tokens;
  uint64_t rows;          // partial rows
};

Cut CutOf(const RoostAmdPagedAttentionF4Params& p, uint32_t cus) {
  Cut c{};
  const uint32_t group = p.q_heads / p.cache.kv_heads;
  c.tiles = group > 16 ? 2 : 1;
  c.short_tokens = 16 * c.tiles / group;
  const uint64_t most = p.kv_indptr.address != nullptr ? p.block_tables.length : p.max_blocks;
  uint64_t keys = p.max_kv_len ? p.max_kv_len : std::min<uint64_t>(most * p.cache.page_size, 16384);
  if (p.window_left >= 0) keys = std::min<uint64_t>(keys, uint64_t{1} * p.window_left + 16 + c.short_tokens);
  keys = std::min<uint64_t>(std::max<uint64_t>(keys, 1), kMostKeys);
  const uint64_t wanted = roost::CeilDiv(4 * cus, std::max<uint64_t>(1, uint64_t{p.batch} * p.cache.kv_heads));
  const uint64_t splits = std::max<uint64_t>(1, std::min<uint64_t>(wanted, roost::CeilDiv(keys, 128)));
  c.part = static_cast<uint32_t>(roost::RoundUp(roost::CeilDiv(keys, splits), 64));
  c.splits = static_cast<uint32_t>(roost::CeilDiv(keys, c.part));
  c.rows = c.splits > 1 ? uint64_t{p.batch} * c.splits * c.short_tokens * p.q_heads : 0;
  return c;
}

uint64_t WorkspaceBytes(const RoostAmdPagedAttentionF4Params& p, uint32_t cus) {
  return CutOf(p, cus).rows * (p.cache.head_dim + 2) * 4;
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

template <int D>
void Launch(const Args& a, const Cut& c, hipStream_t s) {
  const dim3 grid(a.cache.kv_heads, c.splits, a.batch);
  if (c.tiles == 1) {
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
    a.splits = c.splits, a.part = c.part, a.short_tokens = c.short_tokens, a.row_limit = 0x7FFFFFFF;
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
