// GemmLora for gfx950: a projection shared by every sequence, with each sequence's own low-rank adapter and an addend on top.
//
//   y_t = W x_t + scale_a B_a[:, :rank] (A_a[:rank] x_t) + addend_t,   a = the adapter of row t's sequence (or none)
//
// Two launches: ShrinkKernel leaves the low-rank rows u_t = scale_a A_a x_t in the workspace, then the product's kernel
// adds B_a u_t to its own sums before they are stored, so the output is written once.
//
// Operands: everything is moved in 16-byte pieces along the inner dimension (8 bf16, 4 f32 or 16 e4m3). A matrix-instruction
// fragment of 16 rows is one piece a lane: lane l holds row l % 16, piece l / 16 of a 64-byte run. That is the operand layout
// of v_mfma_f32_16x16x32_bf16 as it stands; for f32 (four v_mfma_f32_16x16x4_f32, one word of the piece each) and e4m3 (two
// v_mfma_f32_16x16x32_fp8_fp8, 8 bytes each) the pieces visit the inner dimension in another order, the same for both
// operands, so the sum is over the same products. Weight rows are the first operand and token rows the second: in the result
// lane l holds token l % 16 and the four consecutive outputs 4 (l / 16) .. + 3.

#include <type_traits>

#include "common.h"

namespace {

using namespace roost_dev;

constexpr char kOp[] = "gemm_lora";
constexpr uint32_t kMaxRank = 128;

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

struct E4m3 {
  uint8_t bits;
};

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
  float* u;  // [tokens, max_rank]
  uint64_t x_stride, addend_stride, y_stride;  // elements
  uint32_t tokens, batch, in_dim, out_dim, adapters, max_rank;
  uint32_t addend_f32, y_f32;
};

// ---- Which adapter a row has ---------------------------------------------------------------------------------------

constexpr int32_t kNoRow = -2;      // the row belongs to no sequence
constexpr int32_t kNoAdapter = -1;

// slot[i] for rows t0 .. t0 + n - 1, by the whole workgroup; a barrier must follow.
__device__ __forceinline__ void FillSlots(const LoraArgs& g, uint32_t t0, uint32_t n, int32_t* slot) {
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) slot[i] = kNoRow;
  __syncthreads();
  const auto first = static_cast<int64_t>(t0);
  const int64_t last = min(first + n, static_cast<int64_t>(g.tokens));
  for (uint32_t b = threadIdx.x; b < g.batch; b += blockDim.x) {
    const int64_t lo = max(static_cast<int64_t>(g.cu[b]), first), hi = min(static_cast<int64_t>(g.cu[b + 1]), last);
    if (lo >= hi) continue;
    int32_t s = g.a != nullptr ? g.slots[b] : kNoAdapter;
    if (s < 0 || static_cast<uint32_t>(s) >= g.adapters) s = kNoAdapter;
    for (int64_t t = lo; t < hi; ++t) slot[t - first] = s;
  }
}

__device__ __forceinline__ uint32_t RankOf(const LoraArgs& g, int32_t slot) {
  if (slot < 0) return 0;
  if (g.ranks == nullptr) return g.max_rank;
  return static_cast<uint32_t>(min(max(g.ranks[slot], 0), static_cast<int32_t>(g.max_rank)));
}

// ---- Fragments -------------------------------------------------------------------------------------------------------

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
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u32x2_t pa = {a[2 * i], a[2 * i + 1]}, pb = {b[2 * i], b[2 * i + 1]};
      acc = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(__builtin_bit_cast(long, pa), __builtin_bit_cast(long, pb), acc, 0, 0,
                                                       0);
    }
    return acc;
  }
}

// The piece at byte `at` of a row of `bytes` bytes, zero past its end.
__device__ __forceinline__ u32x4_t Piece(const void* row, uint32_t at, uint32_t bytes) {
  u32x4_t v = {0, 0, 0, 0};
  if (at < bytes) v = *reinterpret_cast<const u32x4_t*>(static_cast<const unsigned char*>(row) + at);
  return v;
}

// Eight e4m3 elements as eight bf16 (exact: e4m3 has three mantissa bits and a smaller exponent range).
__device__ __forceinline__ u32x4_t Bf16OfE4m3(u32x2_t q) {
  u32x4_t v;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(q[i]), false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(q[i]), true);
    v[2 * i] = PackBf16Rne(lo[0], lo[1]);
    v[2 * i + 1] = PackBf16Rne(hi[0], hi[1]);
  }
  return v;
}

// ---- The low-rank rows -------------------------------------------------------------------------------------------------

// Workgroup (i, j, z): rows 16 i .. + 15, ranks 16 j .. + 15, every gridDim.z-th run of rows with one adapter among them.
// Four wavefronts take alternate 64-byte runs of the inner dimension and join their sums through LDS.
template <typename E>
__global__ void __launch_bounds__(256) ShrinkKernel(LoraArgs g) {
  using Low = LowOf<E>;
  __shared__ int32_t slot[16];
  __shared__ f32x4_t part[3][64];
  const uint32_t t0 = 16 * blockIdx.x, r0 = 16 * blockIdx.y;
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  FillSlots(g, t0, 16, slot);
  __syncthreads();
  const uint32_t low_bytes = g.in_dim * sizeof(Low);
  const uint32_t t = min(t0 + lane % 16, g.tokens - 1);
  const E* x = static_cast<const E*>(g.x) + t * g.x_stride;
  uint32_t run = 0;
  for (uint32_t i = 0, next; i < 16; i = next) {
    const int32_t s = slot[i];
    for (next = i + 1; next < 16 && slot[next] == s; ++next) {}
    const uint32_t rank = RankOf(g, s);
    if (r0 >= rank || run++ % gridDim.z != blockIdx.z) continue;
    const Low* a = static_cast<const Low*>(g.a) +
                   (static_cast<uint64_t>(s) * g.max_rank + min(r0 + lane % 16, rank - 1)) * g.in_dim;
    f32x4_t acc = {0, 0, 0, 0};
    for (uint32_t base = 64 * wave; base < low_bytes; base += 256) {
      const uint32_t at = base + 16 * (lane / 16);
      const u32x4_t pa = Piece(a, at, low_bytes);
      u32x4_t px;
      if constexpr (std::is_same_v<E, E4m3>) {
        u32x2_t q = {0, 0};
        if (at < low_bytes) q = *reinterpret_cast<const u32x2_t*>(reinterpret_cast<const unsigned char*>(x) + at / 2);
        px = Bf16OfE4m3(q);
      } else {
        px = Piece(x, at, low_bytes);
      }
      acc = Mma16<Low>(pa, px, acc);
    }
    if (wave > 0) part[wave - 1][lane] = acc;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int w = 0; w < 3; ++w) acc += part[w][lane];
      const uint32_t row = lane % 16;
      float scale = g.lora_scale != nullptr ? g.lora_scale[s] : 1.0f;
      if (row >= i && row < next) {
        if (g.x_scale != nullptr) scale *= g.x_scale[t0 + row];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t r = r0 + 4 * (lane / 16) + e;
          if (r < rank) g.u[static_cast<uint64_t>(t0 + row) * g.max_rank + r] = acc[e] * scale;
        }
      }
    }
    __syncthreads();
  }
}

// ---- The product, straight from memory -----------------------------------------------------------------------------------

// Adds the adapter, the addend and stores four consecutive outputs of one row.
template <typename E>
__device__ __forceinline__ void Finish(const LoraArgs& g, uint32_t t, uint32_t n, int32_t slot, f32x4_t v) {
  using Low = LowOf<E>;
  const uint32_t left = g.out_dim - n;  // outputs from n on
  if constexpr (std::is_same_v<E, E4m3>) {
    const float xs = g.x_scale[t];
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      if (g.w != nullptr && e < left) v[e] *= xs * g.w_scale[n + e];
    }
  }
  const uint32_t rank = RankOf(g, slot);
  const float* u = g.u + static_cast<uint64_t>(t) * g.max_rank;
  for (uint32_t r = 0; r < rank; ++r) {
    const float ur = u[r];
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      if (e < left) {
        const uint64_t at = (static_cast<uint64_t>(slot) * g.out_dim + n + e) * g.max_rank + r;
        float b;
        if constexpr (sizeof(Low) == 2) {
          b = Bf16ToF32(static_cast<const uint16_t*>(g.b)[at]);
        } else {
          b = static_cast<const float*>(g.b)[at];
        }
        v[e] = fmaf(ur, b, v[e]);
      }
    }
  }
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) {
    if (e >= left) continue;
    if (g.addend != nullptr) {
      v[e] += LoadF(g.addend, g.addend_f32 ? ROOST_DTYPE_F32 : ROOST_DTYPE_BF16,
                    static_cast<int64_t>(t * g.addend_stride + n + e));
    }
    const uint64_t at = t * g.y_stride + n + e;
    if (g.y_f32) {
      static_cast<float*>(g.y)[at] = v[e];
    } else {
      static_cast<uint16_t*>(g.y)[at] = F32ToBf16(v[e]);
    }
  }
}

// Workgroup (i, j): outputs 16 i .. + 15 of rows 16 kT j .. + 16 kT - 1. Four wavefronts take alternate 64-byte runs of the
// inner dimension and join their sums through LDS.
template <typename E, int kT>
__global__ void __launch_bounds__(256) ProductKernel(LoraArgs g) {
  __shared__ int32_t slot[16 * kT];
  __shared__ f32x4_t part[4][kT][64];
  const uint32_t n0 = 16 * blockIdx.x, t0 = 16 * kT * blockIdx.y;
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  FillSlots(g, t0, 16 * kT, slot);
  const uint32_t bytes = g.in_dim * sizeof(E);
  f32x4_t acc[kT];
#pragma unroll
  for (int i = 0; i < kT; ++i) acc[i] = f32x4_t{0, 0, 0, 0};
  if (g.w != nullptr) {
    const E* w = static_cast<const E*>(g.w) + static_cast<uint64_t>(min(n0 + lane % 16, g.out_dim - 1)) * g.in_dim;
    const E* x[kT];
#pragma unroll
    for (int i = 0; i < kT; ++i) x[i] = static_cast<const E*>(g.x) + min(t0 + 16 * i + lane % 16, g.tokens - 1) * g.x_stride;
    for (uint32_t base = 64 * wave; base < bytes; base += 256) {
      const uint32_t at = base + 16 * (lane / 16);
      const u32x4_t pw = Piece(w, at, bytes);
#pragma unroll
      for (int i = 0; i < kT; ++i) acc[i] = Mma16<E>(pw, Piece(x[i], at, bytes), acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kT; ++i) part[wave][i][lane] = acc[i];
  __syncthreads();
  for (uint32_t item = threadIdx.x; item < 64 * kT; item += 256) {
    const uint32_t i = item / 64, l = item % 64;
    const uint32_t row = 16 * i + l % 16, n = n0 + 4 * (l / 16);
    const int32_t s = slot[row];
    if (s == kNoRow || n >= g.out_dim) continue;
    f32x4_t v = part[0][i][l];
#pragma unroll
    for (int w = 1; w < 4; ++w) v += part[w][i][l];
    Finish<E>(g, t0 + row, n, s, v);
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

uint64_t WorkspaceBytes(const RoostAmdGemmLoraParams& p) {
  return p.lora_a.address == nullptr ? 0 : static_cast<uint64_t>(p.tokens) * p.max_rank * sizeof(float);
}

// ---- Launch --------------------------------------------------------------------------------------------------------------

template <typename E>
void LaunchAll(const LoraArgs& g, hipStream_t stream) {
  if (g.a != nullptr) {
    const dim3 grid(roost::CeilDiv(g.tokens, 16), roost::CeilDiv(g.max_rank, 16), std::min(std::max(g.batch, 1u), 16u));
    hipLaunchKernelGGL(ShrinkKernel<E>, grid, dim3(256), 0, stream, g);
  }
  const auto product = [&](auto t) {
    constexpr int kT = decltype(t)::value;
    hipLaunchKernelGGL((ProductKernel<E, kT>), dim3(roost::CeilDiv(g.out_dim, 16), roost::CeilDiv(g.tokens, 16 * kT)),
                       dim3(256), 0, stream, g);
  };
  if (g.tokens <= 16) return product(std::integral_constant<int, 1>{});
  return product(std::integral_constant<int, 4>{});
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
    } else {
      LaunchAll<E4m3>(g, s);
    }
    return roost::HipStatus(hipGetLastError(), kOp, "kernel launch");
  });
}
