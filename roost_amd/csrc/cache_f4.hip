// CacheWriteF4 and CacheReadF4 for gfx950: K and V rows into the slots of a 4-bit cache, and back out of them.
//
// Per block of 32 dims: a = max|x|, scale = the smallest power of two with a <= 7 scale, code = e2m1(x / scale). The scale is a
// power of two, so the quotient is exact and the code is the rounding of the value itself: no second rounding anywhere, and any
// other implementation of these three lines gives the same bits. Reading back is exact in bf16 and f32.
//
// Design: memory traffic and, for a step's few rows, one launch's latency. A lane has 8 dims of one head's row (16 bytes of bf16
// in, one word of codes out), so the four lanes of a block share its maximum by two lane swaps and a wavefront reads 1 KB of
// consecutive rows; K and V go in one launch. The scales of a block lie page_size bytes apart per block (their readers' order),
// so each is one byte store; the tokens of a prompt fill a page's lines one behind the other, in L2.
// 8,192 tokens of 8 heads of 128 (42 MB with what is written): 12 us, 3.5 TB/s; a decode step: 1.8 us.

#include "cache_f4.h"

namespace {

using namespace roost_dev;

constexpr uint32_t kThreads = 256;

struct Args {
  void *k, *v;
  uint64_t k_stride, v_stride;  // elements between tokens
  const int64_t* slots;
  roost::CacheF4View cache;
  uint32_t rows;      // tokens x KV heads
  uint32_t vec_shift; // log2(head_dim / 8)
};

// Where 8 dims of one head of one token live: the thread's vector of its row, its slot's page and offset.
struct Place {
  uint32_t token, head, vec;
  uint64_t codes;   // byte of the vector's word
  uint64_t scale;   // byte of its block's scale
  bool live;
};

__device__ __forceinline__ Place PlaceOf(const Args& a) {
  Place p;
  const uint32_t row = (blockIdx.x * (kThreads >> a.vec_shift)) + (threadIdx.x >> a.vec_shift);
  p.vec = threadIdx.x & ((1u << a.vec_shift) - 1);
  p.live = row < a.rows;
  p.token = (p.live ? row : 0) / a.cache.kv_heads;
  p.head = (p.live ? row : 0) - p.token * a.cache.kv_heads;
  const int64_t slot = a.slots[p.token];
  const uint64_t page = static_cast<uint64_t>(slot) >> a.cache.page_shift;
  p.live = p.live && slot >= 0 && page < a.cache.pages;
  const uint64_t offset = static_cast<uint64_t>(slot) & ((1u << a.cache.page_shift) - 1);
  const uint64_t head_page = page * a.cache.kv_heads + p.head;
  p.codes = 4 * ((((head_page << a.cache.page_shift) + offset) << a.vec_shift) + p.vec);
  p.scale = ((((head_page << (a.vec_shift - 2)) + (p.vec >> 2)) << a.cache.page_shift)) + offset;
  return p;
}

typedef uint32_t U4 __attribute__((ext_vector_type(4)));
typedef float F4v __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ void Load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const F4v a = reinterpret_cast<const F4v*>(p)[0], b = reinterpret_cast<const F4v*>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else {
    const U4 w = *reinterpret_cast<const U4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, _Float16>) {
        x[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i])));
        x[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i] >> 16)));
      } else {
        x[2 * i] = Bf16LoToF32(w[i]);
        x[2 * i + 1] = Bf16HiToF32(w[i]);
      }
    }
  }
}

// K's row and V's: both rows' loads go out together.
template <typename T>
__global__ void __launch_bounds__(kThreads) CacheWriteF4Kernel(Args a) {
  const Place p = PlaceOf(a);
  if (!p.live) return;  // whole rows, so a block's four lanes stay together
  const uint64_t at = ((uint64_t{p.head} << a.vec_shift) + p.vec) << 3;
  float x[2][8];
  Load8(static_cast<const T*>(a.k) + p.token * a.k_stride + at, x[0]);
  Load8(static_cast<const T*>(a.v) + p.token * a.v_stride + at, x[1]);
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[v][i]) & 0x7FFFFFFFu);
    // The block's four lanes: a swap of neighbours, then of pairs.
    top = max(top, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(top), 0xB1, 0xf, 0xf, false)));
    top = max(top, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(top), 0x4E, 0xf, 0xf, false)));
    const uint32_t byte = F4ScaleByte(top);
    const uint32_t codes = byte == kF4ByteNan ? 0 : ToF4(x[v], F4Scale(byte));
    *reinterpret_cast<uint32_t*>((v ? a.cache.v : a.cache.k) + p.codes) = codes;
    if ((p.vec & 3) == 0) (v ? a.cache.v_scales : a.cache.k_scales)[p.scale] = static_cast<uint8_t>(byte);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) CacheReadF4Kernel(Args a) {
  const Place p = PlaceOf(a);
  if (!p.live) return;
  const uint64_t at = ((uint64_t{p.head} << a.vec_shift) + p.vec) << 3;
  const uint32_t codes[2] = {*reinterpret_cast<const uint32_t*>(a.cache.k + p.codes),
                             *reinterpret_cast<const uint32_t*>(a.cache.v + p.codes)};
  const float scale[2] = {F4Scale(a.cache.k_scales[p.scale]), F4Scale(a.cache.v_scales[p.scale])};
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    const U4 w{FromF4<0>(codes[v], scale[v]), FromF4<1>(codes[v], scale[v]), FromF4<2>(codes[v], scale[v]),
               FromF4<3>(codes[v], scale[v])};
    T* to = static_cast<T*>(v ? a.v : a.k) + p.token * (v ? a.v_stride : a.k_stride) + at;
    if constexpr (sizeof(T) == 4) {
      U4 lo, hi;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        lo[2 * i] = w[i] << 16, lo[2 * i + 1] = w[i] & 0xFFFF0000u;
        hi[2 * i] = w[2 + i] << 16, hi[2 * i + 1] = w[2 + i] & 0xFFFF0000u;
      }
      reinterpret_cast<U4*>(to)[0] = lo;
      reinterpret_cast<U4*>(to)[1] = hi;
    } else {
      *reinterpret_cast<U4*>(to) = w;
    }
  }
}

RoostStatus Admit(const RoostAmdCacheF4Params& p, const char* op, bool write, uint64_t& pages) {
  roost::Gate gate(op);
  gate.Expect(p.reserved0 == 0, ROOST_STATUS_INVALID_ARGUMENT, "reserved0 = %u, must be 0", p.reserved0);
  roost::AdmitCacheF4(gate, p.cache, pages);
  ROOST_GATE_RETURN(gate);
  const uint32_t dt = p.k.dtype;
  gate.Expect(dt == ROOST_DTYPE_BF16 || dt == ROOST_DTYPE_F32 || (write && dt == ROOST_DTYPE_F16), ROOST_STATUS_UNSUPPORTED,
              "k is %s; rows are bf16, f32%s", roost::Describe(dt).name, write ? " or f16" : " here (f16 cannot hold the range)")
      .Expect(p.tokens < (1u << 24), ROOST_STATUS_UNSUPPORTED, "tokens = %u, not below 2^24", p.tokens)
      .Expect((uint64_t{p.tokens} * p.cache.kv_heads + kThreads) * (p.cache.head_dim / 8) <= 0xFFFFFFFF, ROOST_STATUS_UNSUPPORTED,
              "%u tokens of %u heads of %u exceed one launch's 2^32 threads", p.tokens, p.cache.kv_heads, p.cache.head_dim);
  ROOST_GATE_RETURN(gate);
  if (p.tokens == 0) return ROOST_STATUS_OK;
  const uint64_t width = uint64_t{p.cache.kv_heads} * p.cache.head_dim;
  const uint32_t bytes = roost::ElementBytes(dt);
  const uint64_t ks = p.k_stride ? p.k_stride : width, vs = p.v_stride ? p.v_stride : width;
  gate.Expect(ks >= width && vs >= width, ROOST_STATUS_INVALID_ARGUMENT, "k_stride = %u, v_stride = %u: below a token's %llu",
              p.k_stride, p.v_stride, static_cast<unsigned long long>(width))
      .Expect(ks * bytes % 16 == 0 && vs * bytes % 16 == 0, ROOST_STATUS_INVALID_ARGUMENT,
              "k_stride = %u, v_stride = %u: not multiples of 16 bytes", p.k_stride, p.v_stride)
      .Tensor("k", p.k, dt, (p.tokens - 1) * ks + width)
      .Tensor("v", p.v, dt, (p.tokens - 1) * vs + width)
      .Tensor("slot_mapping", p.slot_mapping, ROOST_DTYPE_I64, p.tokens)
      .Aligned("k", p.k.address, 16)
      .Aligned("v", p.v.address, 16)
      .Aligned("slot_mapping", p.slot_mapping.address, 8);
  ROOST_GATE_RETURN(gate);
  const roost::Extent k = roost::ExtentOf(p.k.address, p.tokens, ks * bytes, width * bytes);
  const roost::Extent v = roost::ExtentOf(p.v.address, p.tokens, vs * bytes, width * bytes);
  const roost::Extent slots = roost::ExtentOf(p.slot_mapping.address, 8 * uint64_t{p.tokens});
  const uint64_t page = uint64_t{p.cache.kv_heads} * p.cache.page_size * p.cache.head_dim / 32;  // bytes of scales
  const roost::Extent cache[] = {
      roost::ExtentOf(p.cache.k.address, pages * page * 16), roost::ExtentOf(p.cache.v.address, pages * page * 16),
      roost::ExtentOf(p.cache.k_scales.address, pages * page), roost::ExtentOf(p.cache.v_scales.address, pages * page)};
  for (int i = 0; i < 4; ++i) {
    for (const auto& other : {k, v, slots}) {
      gate.Expect(!roost::Overlap(cache[i], other), ROOST_STATUS_INVALID_ARGUMENT, "the cache overlaps k, v or slot_mapping");
    }
    for (int j = 0; write && j < i; ++j) {
      gate.Expect(!roost::Overlap(cache[i], cache[j]), ROOST_STATUS_INVALID_ARGUMENT, "spans of the cache overlap");
    }
  }
  gate.Expect(write || (!roost::Overlap(k, v) && !roost::Overlap(k, slots) && !roost::Overlap(v, slots)),
              ROOST_STATUS_INVALID_ARGUMENT, "k, v and slot_mapping overlap");
  return gate.status();
}

RoostStatus Run(RoostContext* ctx, const void* params, void* stream, const char* op, bool write) {
  roost::Gate gate(op);
  gate.Expect(ctx != nullptr, ROOST_STATUS_INVALID_ARGUMENT, "no context was passed").Header(params, sizeof(RoostAmdCacheF4Params));
  ROOST_GATE_RETURN(gate);
  const auto& p = *static_cast<const RoostAmdCacheF4Params*>(params);
  return roost::CatchAll(op, [&]() -> RoostStatus {
    uint64_t pages = 0;
    ROOST_RETURN_IF_FAILED(Admit(p, op, write, pages));
    if (p.tokens == 0) return ROOST_STATUS_OK;
    ROOST_GATE_RETURN(roost::OnDevice(gate, ctx));
    const uint64_t width = uint64_t{p.cache.kv_heads} * p.cache.head_dim;
    Args a{};
    a.k = p.k.address, a.v = p.v.address;
    a.k_stride = p.k_stride ? p.k_stride : width, a.v_stride = p.v_stride ? p.v_stride : width;
    a.slots = static_cast<const int64_t*>(p.slot_mapping.address);
    a.cache = roost::ViewOf(p.cache, pages);
    a.rows = p.tokens * p.cache.kv_heads;
    a.vec_shift = static_cast<uint32_t>(__builtin_ctz(p.cache.head_dim / 8));
    const dim3 grid(static_cast<uint32_t>(roost::CeilDiv(a.rows, kThreads >> a.vec_shift)));
    const hipStream_t s = roost::Stream(stream);
    const bool f32 = p.k.dtype == ROOST_DTYPE_F32;
    if (!write) {
      f32 ? CacheReadF4Kernel<float><<<grid, kThreads, 0, s>>>(a) : CacheReadF4Kernel<uint16_t><<<grid, kThreads, 0, s>>>(a);
    } else if (p.k.dtype == ROOST_DTYPE_F16) {
      CacheWriteF4Kernel<_Float16><<<grid, kThreads, 0, s>>>(a);
    } else {
      f32 ? CacheWriteF4Kernel<float><<<grid, kThreads, 0, s>>>(a) : CacheWriteF4Kernel<uint16_t><<<grid, kThreads, 0, s>>>(a);
    }
    return roost::HipStatus(hipGetLastError(), op, "kernel launch");
  });
}

}  // namespace

extern "C" ROOST_API RoostStatus roost_amd_cache_write_f4_run(RoostContext* ctx, const void* params, void* stream) {
  return Run(ctx, params, stream, "cache_write_f4", true);
}

extern "C" ROOST_API RoostStatus roost_amd_cache_read_f4_run(RoostContext* ctx, const void* params, void* stream) {
  return Run(ctx, params, stream, "cache_read_f4", false);
}
