// The 8-bit paged KV cache (nsa_kv8_cache): geometry, descriptor checks and
// the device arithmetic that its kernels share.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "host_util.h"

namespace nsa {
namespace kv8 {

constexpr int kBlock = 64;       // tokens of a page: one scale per (page, head), K and V apart
constexpr int kRing = 128;       // ring slots: the incomplete block and the one before it
constexpr int kMaxQuery = 64;    // query tokens per call
constexpr int64_t kMaxPos = int64_t(1) << 30;  // positions are 32-bit in the kernels, with room to add to

// Device view of nsa_kv8_cache.
struct Cache {
  int batch, n_kv_heads, n_pages, max_blocks;
  uint8_t *k_codes, *v_codes;
  float2* scales;  // (K, V) of [n_pages, Hkv]
  const int32_t* page_table;
  uint16_t *k_ring, *v_ring;
  int64_t* lens;
  int64_t* ring_floor;
  int32_t* unclean;
  int32_t* tickets;
};

// Strided rows (nsa_kv8_rows) of 16-bit elements.
struct Rows {
  uint16_t* data;
  int64_t sb, sh, st;
  __device__ __forceinline__ uint16_t* row(int64_t b, int64_t h, int64_t t) const {
    return data + b * sb + h * sh + t * st;
  }
};

// Checks a descriptor and fills the device view.
int check_cache(const nsa_kv8_cache* c, Cache& out);
int check_rows(const nsa_kv8_rows* r, const char* name, Rows& out);

// ---------------------------------------------------------------- 16-bit types
template <bool kBf16>
struct Elem;
template <>
struct Elem<false> {
  static constexpr uint32_t kExp = 0x7c007c00u;  // exponent fields of a pair
  __device__ static __forceinline__ float2 unpack(uint32_t x) {
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
  }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) { return pack_half2(lo, hi); }
};
template <>
struct Elem<true> {
  static constexpr uint32_t kExp = 0x7f807f80u;
  __device__ static __forceinline__ float2 unpack(uint32_t x) {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
};
// 0xffff in each half of a pair whose value is not finite.
template <bool kBf16>
__device__ __forceinline__ uint32_t nonfinite_mask(uint32_t x) {
  return __vcmpeq2(x & Elem<kBf16>::kExp, Elem<kBf16>::kExp);
}

}  // namespace kv8
}  // namespace nsa
