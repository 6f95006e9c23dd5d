// AddRmsNorm, AddRmsNormQuant and SiluMulQuant for gfx950: the residual stream's norm in front of a layer's projections,
// and the MLP's activation, both optionally in 8 bits with scales.
//
// Per row, in fp32: s = x + residual (stored, rounded to the residual's type); y = s / sqrt(mean(s^2) + eps) * weight. The
// 8-bit forms cut the row into cells (the whole row, or `group` columns): scale = max(max|y| / 448, 2^-126), code = e4m3(y
// / scale). 448 is e4m3's largest value, so no code overflows; the floor keeps 1 / scale finite for a cell of zeros. The
// quotient is f32's, by the scale's reciprocal and one remainder (quotient.h): 8,192 rows of 12,288 from bf16 take 99.2 us with
// the product by the reciprocal alone, which gives values next to a midpoint the other code, 100.3 so, 104.4 by
// divisions. max|y| is taken over the bit patterns as integers, where a NaN is larger than every number, so a NaN reaches
// the scale instead of being dropped by a float maximum.
//
// Design: pure memory traffic, so one pass: a workgroup holds one row in registers (kV vectors of 8 elements a thread,
// thread t's vector v at column 8 (v * threads + t), so a wavefront reads 1 KB of consecutive bf16), and everything after
// the loads (sum of squares, largest magnitude) is a reduction over registers. A thread's loads of f32 go out one behind
// the other; a bf16 vector is awaited where the branch between whole and short vectors ends, and what hides that is the
// row's other wavefronts. Rows of odd widths or strides take the same path: gfx950 loads 16 bytes from any address that
// suits the element, and only the last few columns of a row, fewer than 8, go one by one.

#include <initializer_list>
#include <type_traits>

#include "common.h"
#include "quotient.h"

namespace {

using namespace roost_dev;

constexpr uint32_t kMaxDim = 32768;  // 4 vectors of 8 columns in each of 1,024 threads
constexpr uint32_t kMaxThreads = 1024;
constexpr float kE4m3Max = 448.0f;
constexpr float kSmallestScale = 1.17549435e-38f;  // 2^-126

// ---- Eight elements of a row ---------------------------------------------------------------------------------------

// Vectors of words at an address that is only aligned to an element.
typedef uint32_t WordsAt1 __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t WordsAt2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t WordsAt4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T>
using WordsOf = std::conditional_t<sizeof(T) == 2, WordsAt2, WordsAt4>;

// Eight consecutive elements as their raw words (4 of bf16, 8 of f32).
template <typename T>
struct Raw8 {
  static constexpr int kWords = sizeof(T) * 2;
  uint32_t w[kWords];
};

// n: the row's elements from p on; past them the words are zero.
template <typename T>
__device__ __forceinline__ void Load8(const T* p, uint32_t n, Raw8<T>& r) {
  typedef WordsOf<T> X4;
  if (n >= 8) {
#pragma unroll
    for (int i = 0; i < Raw8<T>::kWords / 4; ++i) {
      const X4 q = reinterpret_cast<const X4*>(p)[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) r.w[4 * i + j] = q[j];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < Raw8<T>::kWords; ++i) r.w[i] = 0;
#pragma unroll
  for (uint32_t e = 0; e < 7; ++e) {
    if (e < n) {
      if constexpr (sizeof(T) == 2) {
        r.w[e / 2] |= static_cast<uint32_t>(p[e]) << (16 * (e % 2));
      } else {
        r.w[e] = __float_as_uint(p[e]);
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ float Get(const Raw8<T>& r, int e) {
  if constexpr (sizeof(T) == 2) {
    return e % 2 ? Bf16HiToF32(r.w[e / 2]) : Bf16LoToF32(r.w[e / 2]);
  } else {
    return __uint_as_float(r.w[e]);
  }
}

template <typename T>
__device__ __forceinline__ void Store8(T* p, uint32_t n, const float (&v)[8]) {
  typedef WordsOf<T> X4;
  uint32_t w[Raw8<T>::kWords];
#pragma unroll
  for (int i = 0; i < Raw8<T>::kWords; ++i) {
    if constexpr (sizeof(T) == 2) {
      w[i] = PackBf16Rne(v[2 * i], v[2 * i + 1]);
    } else {
      w[i] = __float_as_uint(v[i]);
    }
  }
  if (n >= 8) {
#pragma unroll
    for (int i = 0; i < Raw8<T>::kWords / 4; ++i) {
      reinterpret_cast<X4*>(p)[i] = X4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
    }
    return;
  }
#pragma unroll
  for (uint32_t e = 0; e < 7; ++e) {
    if (e < n) {
      if constexpr (sizeof(T) == 2) {
        p[e] = static_cast<uint16_t>(w[e / 2] >> (16 * (e % 2)));
      } else {
        p[e] = v[e];
      }
    }
  }
}

// Four floats as e4m3 bytes (v_cvt_pk_fp8_f32: round to nearest, ties to even, subnormals kept).
__device__ __forceinline__ uint32_t PackE4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}

// ---- Reductions ------------------------------------------------------------------------------------------------------

__device__ __forceinline__ float WaveSum(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  return v;
}
__device__ __forceinline__ uint32_t WaveMax(uint32_t v, uint32_t lanes) {
  for (uint32_t m = 1; m < lanes; m <<= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), m)));
  return v;
}

// The workgroup's sum, the same bits in every thread (each adds the wavefronts' sums in the same order).
__device__ __forceinline__ float BlockSum(float v, float* lds) {
  const uint32_t waves = blockDim.x / 64;
  v = WaveSum(v);
  if (waves == 1) return v;
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
  __syncthreads();
  float sum = 0.0f;
  for (uint32_t i = 0; i < waves; ++i) sum += lds[i];
  return sum;
}
__device__ __forceinline__ uint32_t BlockMax(uint32_t v, uint32_t* lds) {
  const uint32_t waves = blockDim.x / 64;
  v = WaveMax(v, 64);
  if (waves == 1) return v;
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
  __syncthreads();
  uint32_t top = 0;
  for (uint32_t i = 0; i < waves; ++i) top = max(top, lds[i]);
  return top;
}

// ---- 8 bits and scales -----------------------------------------------------------------------------------------------

struct QuantArgs {
  uint8_t* y;
  float* scales;
  uint64_t y_stride;
  uint32_t dim, group;  // group 0: one cell a row
  uint32_t cells;       // of a row
};

// Writes a row's values y[v][e] (zero past the row's end) as codes and scales.
template <int kV>
__device__ __forceinline__ void StoreQuantised(const QuantArgs& a, uint64_t row, const float (&y)[kV][8]) {
  __shared__ uint32_t lds[kMaxThreads / 64];
  uint32_t top[kV];
#pragma unroll
  for (int v = 0; v < kV; ++v) {
    top[v] = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top[v] = max(top[v], __float_as_uint(y[v][e]) & 0x7FFFFFFFu);
  }
  if (a.group == 0) {
    uint32_t t = top[0];
#pragma unroll
    for (int v = 1; v < kV; ++v) t = max(t, top[v]);
    t = BlockMax(t, lds);
#pragma unroll
    for (int v = 0; v < kV; ++v) top[v] = t;
  } else {
    // A cell is group / 8 neighbouring lanes: a power of two up to 64, and the row's vectors start at lane 0.
#pragma unroll
    for (int v = 0; v < kV; ++v) top[v] = WaveMax(top[v], a.group / 8);
  }
#pragma unroll
  for (int v = 0; v < kV; ++v) {
    const uint32_t c = 8 * (v * blockDim.x + threadIdx.x);
    if (c >= a.dim) continue;
    float scale = __fdiv_rn(__uint_as_float(top[v]), kE4m3Max);
    if (scale < kSmallestScale) scale = kSmallestScale;  // false for a NaN, which stays
    if (a.group == 0 ? c == 0 : c % a.group == 0) a.scales[row * a.cells + (a.group ? c / a.group : 0)] = scale;
    float q[8];
    if (scale >= roost::kQuotientLow && scale <= roost::kQuotientHigh) {
      const float inverse = __fdiv_rn(1.0f, scale);
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = roost::Quotient(y[v][e], scale, inverse);
    } else {  // next to f32's ends, infinite or NaN
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = __fdiv_rn(y[v][e], scale);
    }
    const uint32_t w[2] = {PackE4m3(q[0], q[1], q[2], q[3]), PackE4m3(q[4], q[5], q[6], q[7])};
    uint8_t* p = a.y + row * a.y_stride + c;
    if (a.dim - c >= 8) {
      *reinterpret_cast<WordsAt1*>(p) = WordsAt1{w[0], w[1]};
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 7; ++e) {
        if (e < a.dim - c) p[e] = static_cast<uint8_t>(w[e / 4] >> (8 * (e % 4)));
      }
    }
  }
}

// ---- AddRmsNorm and AddRmsNormQuant ------------------------------------------------------------------------------------

struct NormArgs {
  const void *x, *residual, *weight;
  void *residual_out, *y;
  uint64_t x_stride, residual_stride, residual_out_stride, y_stride;
  uint32_t dim;
  float eps;
  QuantArgs quant;
};

// TX, TR, TW: the types of the input, the residual and the weight; kQuant: 8-bit output. One workgroup a row.
template <typename TX, typename TR, typename TW, bool kQuant, int kV>
__global__ void __launch_bounds__(kMaxThreads) AddRmsNormKernel(NormArgs a) {
  __shared__ float lds[kMaxThreads / 64];
  const uint64_t row = blockIdx.x;
  const TX* x = static_cast<const TX*>(a.x) + row * a.x_stride;
  const TR* res = static_cast<const TR*>(a.residual) + row * a.residual_stride;
  Raw8<TX> rx[kV];
  Raw8<TR> rr[kV];
#pragma unroll
  for (int v = 0; v < kV; ++v) {
    const uint32_t c = 8 * (v * blockDim.x + threadIdx.x);
    const uint32_t n = c < a.dim ? a.dim - c : 0;
    Load8(x + c, n, rx[v]);
    if (a.residual != nullptr) Load8(res + c, n, rr[v]);
  }
  Raw8<TW> rw[kV];
#pragma unroll
  for (int v = 0; v < kV; ++v) {
    const uint32_t c = 8 * (v * blockDim.x + threadIdx.x);
    const uint32_t n = c < a.dim ? a.dim - c : 0;
    Load8(static_cast<const TW*>(a.weight) + c, n, rw[v]);
  }
  float s[kV][8];
  float sum = 0.0f;
#pragma unroll
  for (int v = 0; v < kV; ++v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      s[v][e] = Get(rx[v], e);
      if (a.residual != nullptr) s[v][e] += Get(rr[v], e);
      sum = fmaf(s[v][e], s[v][e], sum);
    }
  }
  if (a.residual_out != nullptr) {
    TR* out = static_cast<TR*>(a.residual_out) + row * a.residual_out_stride;
#pragma unroll
    for (int v = 0; v < kV; ++v) {
      const uint32_t c = 8 * (v * blockDim.x + threadIdx.x);
      if (c < a.dim) Store8(out + c, a.dim - c, s[v]);
    }
  }
  const float mean = __fdiv_rn(BlockSum(sum, lds), static_cast<float>(a.dim));
  const float r = __fdiv_rn(1.0f, __fsqrt_rn(mean + a.eps));
#pragma unroll
  for (int v = 0; v < kV; ++v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s[v][e] = s[v][e] * r * Get(rw[v], e);
  }
  if constexpr (kQuant) {
    // Columns past the row's end hold 0 * r * 0: a NaN where r is not finite, which must not reach the cell's maximum.
#pragma unroll
    for (int v = 0; v < kV; ++v) {
      const uint32_t c = 8 * (v * blockDim.x + threadIdx.x);
#pragma unroll
      for (uint32_t e = 0; e < 8; ++e) s[v][e] = c + e < a.dim ? s[v][e] : 0.0f;
    }
    StoreQuantised(a.quant, row, s);
  } else {
    TX* y = static_cast<TX*>(a.y) + row * a.y_stride;
#pragma unroll
    for (int v = 0; v < kV; ++v) {
      const uint32_t c = 8 * (v * blockDim.x + threadIdx.x);
      if (c < a.dim) Store8(y + c, a.dim - c, s[v]);
    }
  }
}

// ---- SiluMulQuant ------------------------------------------------------------------------------------------------------

struct SiluArgs {
  const void *gate, *up;
  uint64_t gate_stride, up_stride;
  QuantArgs quant;
};

template <typename T, int kV>
__global__ void __launch_bounds__(kMaxThreads) SiluMulQuantKernel(SiluArgs a) {
  const uint64_t row = blockIdx.x;
  const T* gate = static_cast<const T*>(a.gate) + row * a.gate_stride;
  const T* up = static_cast<const T*>(a.up) + row * a.up_stride;
  Raw8<T> rg[kV], ru[kV];
#pragma unroll
  for (int v = 0; v < kV; ++v) {
    const uint32_t c = 8 * (v * blockDim.x + threadIdx.x);
    const uint32_t n = c < a.quant.dim ? a.quant.dim - c : 0;
    Load8(gate + c, n, rg[v]);
    Load8(up + c, n, ru[v]);
  }
  float y[kV][8];
#pragma unroll
  for (int v = 0; v < kV; ++v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[v][e] = SiluF(Get(rg[v], e)) * Get(ru[v], e);
  }
  StoreQuantised(a.quant, row, y);
}

// ---- Admission -----------------------------------------------------------------------------------------------------------

bool FloatType(uint32_t dt) { return dt == ROOST_DTYPE_BF16 || dt == ROOST_DTYPE_F32; }

// The bytes a span of rows covers.
struct Rows {
  uintptr_t first = 0;
  uint64_t rows = 0, width = 0, stride = 0;  // bytes
  uint32_t dtype = 0;
  uintptr_t end() const { return first + (rows - 1) * stride + width; }
};
Rows RowsOf(const RoostDeviceSpan& s, uint64_t rows, uint64_t dim, uint64_t stride) {
  const uint64_t e = roost::ElementBytes(s.dtype);
  return Rows{reinterpret_cast<uintptr_t>(s.address), rows, dim * e, stride * e, s.dtype};
}
// Whether two spans share a byte. Rows of the same stride may lie side by side (column views of one tensor).
bool Overlap(const Rows& a, const Rows& b) {
  if (a.first == 0 || b.first == 0 || a.rows == 0 || b.rows == 0) return false;
  if (!(a.first < b.end() && b.first < a.end())) return false;
  if (a.stride != b.stride || a.stride == 0) return true;
  const uint64_t off = b.first >= a.first ? (b.first - a.first) % a.stride  // b's column in a's rows
                                          : (a.stride - (a.first - b.first) % a.stride) % a.stride;
  return off < a.width || off + b.width > a.stride;
}
bool Same(const Rows& a, const Rows& b) {
  return a.first == b.first && a.stride == b.stride && a.dtype == b.dtype;
}

uint64_t StrideOr(uint32_t stride, uint32_t dim) { return stride == 0 ? dim : stride; }

// A [rows, dim] span at `stride` elements a row, of the type `dtype`.
roost::Gate& RowSpan(roost::Gate& gate, const char* name, const RoostDeviceSpan& s, uint32_t dtype, uint32_t rows,
                     uint32_t dim, uint32_t stride) {
  gate.Expect(stride == 0 || stride >= dim, ROOST_STATUS_INVALID_ARGUMENT, "%s: row stride %u below dim = %u", name, stride,
              dim);
  if (!gate.ok()) return gate;
  const uint64_t need = rows == 0 ? 0 : (rows - 1ull) * StrideOr(stride, dim) + dim;
  return gate.Tensor(name, s, dtype, need).Aligned(name, s.address, roost::ElementBytes(dtype));
}

// Vectors a thread holds and threads of a row's workgroup: one vector a thread as long as the row's threads fit a
// workgroup, for more of a row's wavefronts hide more of each other's waits. Against 2 and 4 a thread: 8,192 rows of 4,096
// bf16 onto f32 70.9 and 75.9 us, 64 rows of 4,096 to e4m3 4.1 and 5.0 us, 6,007 rows of 5,000 to e4m3 by groups 49 and 58
// us (4 a thread).
struct Shape {
  int per_thread;
  uint32_t threads;
};
Shape ShapeOf(uint32_t dim) {
  const uint64_t vectors = roost::CeilDiv(dim, 8);
  const int v = vectors <= kMaxThreads ? 1 : vectors <= 2 * kMaxThreads ? 2 : 4;
  return Shape{v, static_cast<uint32_t>(roost::RoundUp(roost::CeilDiv(vectors, v), 64))};
}

roost::Gate& Size(roost::Gate& gate, uint32_t rows, uint32_t dim) {
  gate.Expect(dim > 0 && dim <= kMaxDim, ROOST_STATUS_UNSUPPORTED, "dim = %u; built for 1 to %u columns", dim, kMaxDim);
  if (!gate.ok()) return gate;
  return gate.Expect(uint64_t{rows} * ShapeOf(dim).threads < 1ull << 32, ROOST_STATUS_UNSUPPORTED,
                     "rows = %u of %u columns; a launch is below 2^32 threads, %u to a row", rows, dim, ShapeOf(dim).threads);
}

roost::Gate& Quant(roost::Gate& gate, const RoostDeviceSpan& y, const RoostDeviceSpan& scales, uint32_t rows, uint32_t dim,
                   uint32_t y_stride, uint32_t group) {
  gate.Expect(group == 0 || (group >= 16 && group <= 512 && roost::IsPow2(group)), ROOST_STATUS_UNSUPPORTED,
              "group_size = %u; built for 0 (a scale for each row) and powers of two from 16 to 512", group);
  if (!gate.ok()) return gate;
  RowSpan(gate, "output", y, ROOST_DTYPE_F8E4M3, rows, dim, y_stride);
  const uint64_t cells = group == 0 ? 1 : roost::CeilDiv(dim, group);
  return gate.Tensor("scales", scales, ROOST_DTYPE_F32, rows * cells).Aligned("scales", scales.address, 4);
}

QuantArgs MakeQuant(const RoostDeviceSpan& y, const RoostDeviceSpan& scales, uint32_t dim, uint32_t y_stride,
                    uint32_t group) {
  return QuantArgs{static_cast<uint8_t*>(y.address), static_cast<float*>(scales.address), StrideOr(y_stride, dim), dim, group,
                   group == 0 ? 1u : static_cast<uint32_t>(roost::CeilDiv(dim, group))};
}

// The rules the two norms share; `p` is either params struct.
template <typename Params>
void AdmitNorm(roost::Gate& gate, const Params& p, uint32_t out_type) {
  Size(gate, p.rows, p.dim)
      .Expect(FloatType(p.input.dtype), ROOST_STATUS_UNSUPPORTED, "input is %s; built for bf16 and f32",
              roost::Describe(p.input.dtype).name)
      .Expect(FloatType(p.weight.dtype), ROOST_STATUS_UNSUPPORTED, "weight is %s; built for bf16 and f32",
              roost::Describe(p.weight.dtype).name);
  if (!gate.ok()) return;
  const bool has_res = p.residual.address != nullptr, has_out = p.residual_out.address != nullptr;
  const uint32_t res_type = has_res ? p.residual.dtype : p.input.dtype;
  gate.Expect(FloatType(res_type), ROOST_STATUS_UNSUPPORTED, "residual is %s; built for bf16 and f32",
              roost::Describe(res_type).name);
  if (!gate.ok()) return;
  RowSpan(gate, "input", p.input, p.input.dtype, p.rows, p.dim, p.input_stride);
  if (gate.ok() && has_res) RowSpan(gate, "residual", p.residual, res_type, p.rows, p.dim, p.residual_stride);
  if (gate.ok() && has_out) RowSpan(gate, "residual_out", p.residual_out, res_type, p.rows, p.dim, p.residual_out_stride);
  if (!gate.ok()) return;
  gate.Tensor("weight", p.weight, p.weight.dtype, p.dim)
      .Aligned("weight", p.weight.address, roost::ElementBytes(p.weight.dtype));
  if (!gate.ok()) return;
  const Rows x = RowsOf(p.input, p.rows, p.dim, StrideOr(p.input_stride, p.dim));
  const Rows r = has_res ? RowsOf(p.residual, p.rows, p.dim, StrideOr(p.residual_stride, p.dim)) : Rows{};
  const Rows ro = has_out ? RowsOf(p.residual_out, p.rows, p.dim, StrideOr(p.residual_out_stride, p.dim)) : Rows{};
  RoostDeviceSpan out = p.output;
  out.dtype = out_type;
  const Rows y = RowsOf(out, p.rows, p.dim, StrideOr(p.output_stride, p.dim));
  const Rows w = RowsOf(p.weight, 1, p.dim, p.dim);
  const auto clash = [](const Rows& out_rows, const Rows& in) { return Overlap(out_rows, in) && !Same(out_rows, in); };
  gate.Expect(!clash(y, x) && !clash(y, r) && !clash(ro, x) && !clash(ro, r), ROOST_STATUS_INVALID_ARGUMENT,
              "output or residual_out overlaps input or residual without being exactly that span")
      .Expect(!Overlap(y, ro) && !Overlap(y, w) && !Overlap(ro, w), ROOST_STATUS_INVALID_ARGUMENT,
              "output, residual_out and weight overlap");
}

bool ScalesClash(const RoostDeviceSpan& scales, uint64_t count, std::initializer_list<Rows> others) {
  const Rows s = RowsOf(scales, 1, count, count);
  for (const Rows& o : others) {
    if (Overlap(s, o)) return true;
  }
  return false;
}

// ---- Launch --------------------------------------------------------------------------------------------------------------

// Calls f with the number of vectors as a constant.
template <typename F>
void WithVectors(int v, F&& f) {
  if (v == 1) return f(std::integral_constant<int, 1>{});
  if (v == 2) return f(std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, 4>{});
}
template <typename F>
void WithFloat(uint32_t dtype, F&& f) {
  if (dtype == ROOST_DTYPE_F32) return f(float{});
  return f(uint16_t{});
}

template <bool kQuant, typename Params>
RoostStatus LaunchNorm(const Params& p, const QuantArgs& quant, hipStream_t stream, const char* op) {
  NormArgs a{};
  a.x = p.input.address, a.residual = p.residual.address, a.weight = p.weight.address;
  a.residual_out = p.residual_out.address, a.y = p.output.address;
  a.x_stride = StrideOr(p.input_stride, p.dim), a.residual_stride = StrideOr(p.residual_stride, p.dim);
  a.residual_out_stride = StrideOr(p.residual_out_stride, p.dim), a.y_stride = StrideOr(p.output_stride, p.dim);
  a.dim = p.dim, a.eps = p.eps, a.quant = quant;
  const Shape shape = ShapeOf(p.dim);
  const uint32_t res_type = p.residual.address != nullptr ? p.residual.dtype : p.input.dtype;
  WithFloat(p.input.dtype, [&](auto x) {
    WithFloat(res_type, [&](auto r) {
      WithFloat(p.weight.dtype, [&](auto w) {
        WithVectors(shape.per_thread, [&](auto v) {
          hipLaunchKernelGGL((AddRmsNormKernel<decltype(x), decltype(r), decltype(w), kQuant, decltype(v)::value>),
                             dim3(p.rows), dim3(shape.threads), 0, stream, a);
        });
      });
    });
  });
  return roost::HipStatus(hipGetLastError(), op, "kernel launch");
}

}  // namespace

extern "C" ROOST_API RoostStatus roost_amd_add_rms_norm_run(RoostContext* ctx, const void* params, void* stream) {
  constexpr char kOp[] = "add_rms_norm";
  roost::Gate gate(kOp);
  gate.Expect(ctx != nullptr, ROOST_STATUS_INVALID_ARGUMENT, "no context was passed")
      .Header(params, sizeof(RoostAmdAddRmsNormParams));
  ROOST_GATE_RETURN(gate);
  const auto& p = *static_cast<const RoostAmdAddRmsNormParams*>(params);
  return roost::CatchAll(kOp, [&]() -> RoostStatus {
    gate.Expect(p.reserved0 == 0, ROOST_STATUS_INVALID_ARGUMENT, "reserved0 = %u, must be 0", p.reserved0);
    AdmitNorm(gate, p, p.input.dtype);
    ROOST_GATE_RETURN(gate);
    RowSpan(gate, "output", p.output, p.input.dtype, p.rows, p.dim, p.output_stride);
    ROOST_GATE_RETURN(gate);
    if (p.rows == 0) return ROOST_STATUS_OK;
    ROOST_GATE_RETURN(roost::OnDevice(gate, ctx));
    return LaunchNorm<false>(p, QuantArgs{}, roost::Stream(stream), kOp);
  });
}

extern "C" ROOST_API RoostStatus roost_amd_add_rms_norm_quant_run(RoostContext* ctx, const void* params, void* stream) {
  constexpr char kOp[] = "add_rms_norm_quant";
  roost::Gate gate(kOp);
  gate.Expect(ctx != nullptr, ROOST_STATUS_INVALID_ARGUMENT, "no context was passed")
      .Header(params, sizeof(RoostAmdAddRmsNormQuantParams));
  ROOST_GATE_RETURN(gate);
  const auto& p = *static_cast<const RoostAmdAddRmsNormQuantParams*>(params);
  return roost::CatchAll(kOp, [&]() -> RoostStatus {
    AdmitNorm(gate, p, ROOST_DTYPE_F8E4M3);
    ROOST_GATE_RETURN(gate);
    Quant(gate, p.output, p.scales, p.rows, p.dim, p.output_stride, p.group_size);
    ROOST_GATE_RETURN(gate);
    const QuantArgs quant = MakeQuant(p.output, p.scales, p.dim, p.output_stride, p.group_size);
    gate.Expect(!ScalesClash(p.scales, uint64_t{p.rows} * quant.cells,
                             {RowsOf(p.input, p.rows, p.dim, StrideOr(p.input_stride, p.dim)),
                              RowsOf(p.residual, p.rows, p.dim, StrideOr(p.residual_stride, p.dim)),
                              RowsOf(p.residual_out, p.rows, p.dim, StrideOr(p.residual_out_stride, p.dim)),
                              RowsOf(p.output, p.rows, p.dim, StrideOr(p.output_stride, p.dim)),
                              RowsOf(p.weight, 1, p.dim, p.dim)}),
                ROOST_STATUS_INVALID_ARGUMENT, "scales overlap another span of the call");
    ROOST_GATE_RETURN(gate);
    if (p.rows == 0) return ROOST_STATUS_OK;
    ROOST_GATE_RETURN(roost::OnDevice(gate, ctx));
    return LaunchNorm<true>(p, quant, roost::Stream(stream), kOp);
  });
}

extern "C" ROOST_API RoostStatus roost_amd_silu_mul_quant_run(RoostContext* ctx, const void* params, void* stream) {
  constexpr char kOp[] = "silu_mul_quant";
  roost::Gate gate(kOp);
  gate.Expect(ctx != nullptr, ROOST_STATUS_INVALID_ARGUMENT, "no context was passed")
      .Header(params, sizeof(RoostAmdSiluMulQuantParams));
  ROOST_GATE_RETURN(gate);
  const auto& p = *static_cast<const RoostAmdSiluMulQuantParams*>(params);
  return roost::CatchAll(kOp, [&]() -> RoostStatus {
    Size(gate, p.rows, p.dim)
        .Expect(FloatType(p.gate.dtype), ROOST_STATUS_UNSUPPORTED, "gate is %s; built for bf16 and f32",
                roost::Describe(p.gate.dtype).name);
    ROOST_GATE_RETURN(gate);
    RowSpan(gate, "gate", p.gate, p.gate.dtype, p.rows, p.dim, p.gate_stride);
    RowSpan(gate, "up", p.up, p.gate.dtype, p.rows, p.dim, p.up_stride);
    Quant(gate, p.output, p.scales, p.rows, p.dim, p.output_stride, p.group_size);
    ROOST_GATE_RETURN(gate);
    SiluArgs a{p.gate.address, p.up.address, StrideOr(p.gate_stride, p.dim), StrideOr(p.up_stride, p.dim),
               MakeQuant(p.output, p.scales, p.dim, p.output_stride, p.group_size)};
    const Rows g = RowsOf(p.gate, p.rows, p.dim, a.gate_stride), u = RowsOf(p.up, p.rows, p.dim, a.up_stride);
    const Rows y = RowsOf(p.output, p.rows, p.dim, a.quant.y_stride);
    gate.Expect(!Overlap(y, g) && !Overlap(y, u) && !ScalesClash(p.scales, uint64_t{p.rows} * a.quant.cells, {g, u, y}),
                ROOST_STATUS_INVALID_ARGUMENT, "output or scales overlap another span of the call");
    ROOST_GATE_RETURN(gate);
    if (p.rows == 0) return ROOST_STATUS_OK;
    ROOST_GATE_RETURN(roost::OnDevice(gate, ctx));
    const Shape shape = ShapeOf(p.dim);
    WithFloat(p.gate.dtype, [&](auto t) {
      WithVectors(shape.per_thread, [&](auto v) {
        hipLaunchKernelGGL((SiluMulQuantKernel<decltype(t), decltype(v)::value>), dim3(p.rows), dim3(shape.threads), 0,
                           roost::Stream(stream), a);
      });
    });
    return roost::HipStatus(hipGetLastError(), kOp, "kernel launch");
  });
}
