// Writing tokens into the 8-bit paged cache and reading them back.
//
// Append: a block X of 64 tokens and one head becomes
//   s = max(max|X| / top, 2^-126),  c = round(X * (1/s)),  value = s * c.
// The multiplication by the rounded reciprocal is part of the definition (it
// moves a code only where X/s lies within 2^-23 of a rounding border); float32
// throughout, so the codes are reproducible to the bit.  Bound by HBM: 2 bytes
// in and 1 byte out per element.  One CTA holds a whole block of K and of V in
// registers (8 K + 8 V elements a thread and row), so the tokens are read once
// for both the maximum and the codes.  16 prompts of 8000 tokens, 8 heads of 128,
// bf16: 127 us, 0.95 of the measured copy rate.

#include "kv8.cuh"

namespace nsa {
namespace kv8 {

int check_cache(const nsa_kv8_cache* c, Cache& out) {
  if (!c) return fail(NSA_ERR_INVALID, "cache descriptor is NULL");
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(NSA_ERR_UNSUPPORTED, "head_dim must be 64 or 128, got %lld", (long long)c->head_dim);
  if (c->dtype != 1 && c->dtype != 2) return fail(NSA_ERR_UNSUPPORTED, "dtype must be 1 (float16) or 2 (bfloat16)");
  if (c->codes != NSA_KV8_E4M3 && c->codes != NSA_KV8_INT8)
    return fail(NSA_ERR_UNSUPPORTED, "codes must be NSA_KV8_E4M3 or NSA_KV8_INT8");
  if (c->batch < 0 || c->n_kv_heads < 1 || c->n_pages < 1 || c->max_blocks < 1)
    return fail(NSA_ERR_INVALID, "need batch >= 0 and n_kv_heads, n_pages, max_blocks >= 1");
  if (c->max_blocks * kBlock > kMaxPos || c->batch > (1 << 20) || c->n_kv_heads > (1 << 16) ||
      c->batch * c->n_kv_heads > (1 << 23))
    return fail(NSA_ERR_UNSUPPORTED, "at most 2^30 tokens a sequence, 2^20 sequences and 2^23 (sequence, head) pairs");
  // rows of the tensor maps are 32-bit coordinates
  if (c->n_pages > (int64_t(1) << 31) / (c->n_kv_heads * kBlock) - 1)
    return fail(NSA_ERR_UNSUPPORTED, "n_pages * n_kv_heads * 64 must stay below 2^31");
  if (!c->k_codes || !c->v_codes || !c->scales ||
      (c->batch > 0 && (!c->page_table || !c->k_ring || !c->v_ring || !c->lens || !c->ring_floor || !c->unclean || !c->tickets)))
    return fail(NSA_ERR_INVALID, "null pointer in the cache descriptor");
  if (!aligned16(c->k_codes) || !aligned16(c->v_codes) || !aligned16(c->k_ring) || !aligned16(c->v_ring) ||
      !aligned16(c->scales))
    return fail(NSA_ERR_ALIGN, "codes, scales and rings must be 16-byte aligned");
  out.batch = static_cast<int>(c->batch);
  out.n_kv_heads = static_cast<int>(c->n_kv_heads);
  out.n_pages = static_cast<int>(c->n_pages);
  out.max_blocks = static_cast<int>(c->max_blocks);
  out.k_codes = static_cast<uint8_t*>(c->k_codes);
  out.v_codes = static_cast<uint8_t*>(c->v_codes);
  out.scales = reinterpret_cast<float2*>(c->scales);
  out.page_table = c->page_table;
  out.k_ring = static_cast<uint16_t*>(c->k_ring);
  out.v_ring = static_cast<uint16_t*>(c->v_ring);
  out.lens = c->lens;
  out.ring_floor = c->ring_floor;
  out.unclean = c->unclean;
  out.tickets = c->tickets;
  return NSA_OK;
}

int check_rows(const nsa_kv8_rows* r, const char* name, Rows& out) {
  if (!r || !r->data) return fail(NSA_ERR_INVALID, "%s is NULL", name);
  if (!aligned16(r->data) || ((r->batch_stride | r->head_stride | r->token_stride) & 7))
    return fail(NSA_ERR_ALIGN, "rows of %s must be 16-byte aligned (strides multiples of 8 elements)", name);
  out.data = static_cast<uint16_t*>(r->data);
  out.sb = r->batch_stride;
  out.sh = r->head_stride;
  out.st = r->token_stride;
  return NSA_OK;
}

namespace {

constexpr int kThreads = 256;

struct AppendParams {
  Cache c;
  Rows k, v;
  int n_tokens;
  const int64_t* starts;
  const int64_t* counts;
  int* err;
};

// ring_floor[b] holds the oldest position of which the ring has the tokens, and
// the length that an append or adoption left: the ring is known to reach back that
// far as long as the sequence still has this length.  One that got another by a
// write to lens (pages of a shared prefix) has its incomplete block there at most.
__device__ __forceinline__ int64_t ring_state(int64_t floor, int64_t len) { return floor | (len << 32); }
__device__ __forceinline__ int64_t ring_reach(int64_t state, int64_t len) {
  return (state >> 32) == len ? (state & 0xffffffff) : len / kBlock * kBlock;
}

// Where a sequence's new tokens go; ok = 0 leaves it as it was.
struct Span {
  int start, end, ok;
  int anew;  // the ring holds nothing of the tokens before
};

// max(m, |x|) over the 8 elements of x; NaN stays.
__device__ __forceinline__ void amax8(const uint4& x, __half2& m) {
  const __half2* h = reinterpret_cast<const __half2*>(&x);
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __hmax2_nan(m, __habs2(h[i]));
}
__device__ __forceinline__ void amax8(const uint4& x, __nv_bfloat162& m) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&x);
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __hmax2_nan(m, __habs2(h[i]));
}
template <bool kBf16, int N>
__device__ __forceinline__ float amax_of(const uint4 (&x)[N]) {
  float a, b;
  if constexpr (kBf16) {
    __nv_bfloat162 m = __float2bfloat162_rn(0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) amax8(x[i], m);
    a = __low2float(m), b = __high2float(m);
  } else {
    __half2 m = __float2half2_rn(0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) amax8(x[i], m);
    a = __low2float(m), b = __high2float(m);
  }
  // a value that is not finite counts as infinity from here on
  const float y = (a < INFINITY) ? a : INFINITY, z = (b < INFINITY) ? b : INFINITY;
  return fmaxf(y, z);
}

template <bool kInt8>
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d) {
  if constexpr (kInt8) {
    const int i = __float2int_rn(fminf(fmaxf(a, -127.f), 127.f)), j = __float2int_rn(fminf(fmaxf(b, -127.f), 127.f));
    const int k = __float2int_rn(fminf(fmaxf(c, -127.f), 127.f)), l = __float2int_rn(fminf(fmaxf(d, -127.f), 127.f));
    return (i & 255) | ((j & 255) << 8) | ((k & 255) << 16) | (static_cast<uint32_t>(l) << 24);
  } else {  // the conversion saturates at 448
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return lo | (static_cast<uint32_t>(hi) << 16);
  }
}

template <bool kBf16, bool kInt8>
__device__ __forceinline__ uint2 codes8(const uint4& x, float inv) {
  const float2 a = Elem<kBf16>::unpack(x.x), b = Elem<kBf16>::unpack(x.y), c = Elem<kBf16>::unpack(x.z),
               d = Elem<kBf16>::unpack(x.w);
  uint2 r;
  r.x = code4<kInt8>(a.x * inv, a.y * inv, b.x * inv, b.y * inv);
  r.y = code4<kInt8>(c.x * inv, c.y * inv, d.x * inv, d.y * inv);
  return r;
}

__device__ __forceinline__ uint4 ldg16(const uint16_t* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

// One thread of every CTA asks for its unit's span; the last of a sequence's
// `askers` to have read its length sets the new one.
__device__ __forceinline__ Span take_span(const AppendParams& p, int b, int askers) {
  const Cache& c = p.c;
  const int64_t len = c.lens[b], cap = int64_t(c.max_blocks) * kBlock,
                floor = ring_reach(c.ring_floor[b], len);
  const int64_t s = p.starts ? p.starts[b] : len;
  const int64_t n = p.counts ? p.counts[b] : p.n_tokens;
  const bool ok = s >= 0 && s <= len && len <= cap && n >= 0 && n <= p.n_tokens && s + n <= cap &&
                  (s % kBlock == 0 || s >= floor);
  if (!ok) set_error(p.err, NSA_ERR_INVALID);
  const bool anew = ok && s <= floor;
  // The ticket's step is made from `ok` and `anew` (the same for all of a sequence's
  // askers): it cannot be taken before what this thread needs of lens and floor is there.
  // That is an order of the machine, which does not guess the operand of an atomic;
  // the memory model would ask for a release, which costs 7 us in a prompt of 8000
  // tokens (129 us) and 0.8 in a step of 256 sequences.
  const unsigned step = anew ? 1 : ok ? 2 : 3;
  if (atomicAdd(reinterpret_cast<unsigned*>(c.tickets + b), step) == (askers - 1) * step) {
    c.tickets[b] = 0;
    if (ok) {
      const int64_t first = s / kBlock * kBlock, last = (s + n) / kBlock * kBlock;
      c.lens[b] = s + n;
      c.ring_floor[b] = ring_state(max(s < floor ? first : floor, last - kBlock), s + n);
    }
  }
  return Span{ok ? static_cast<int>(s) : 0, ok ? static_cast<int>(s + n) : 0, ok, anew};
}

// Quantizes block i of a unit, which a whole CTA calls for: its tokens from
// the ring up to `start`, from the new tokens on.
template <int kD, bool kBf16, bool kInt8>
__device__ __forceinline__ void quantize_block(const AppendParams& p, int b, int h, int i, int start, int tid,
                                               float2* red) {
  constexpr int kVecs = kD / 8;                // 16-byte vectors a row
  constexpr int kRowsPass = kThreads / kVecs;  // rows a pass
  constexpr int kN = kBlock / kRowsPass;       // vectors a thread of K (and of V)
  const Cache& c = p.c;
  const int col = (tid % kVecs) * 8, row0 = tid / kVecs;
  const int64_t ring = (int64_t(b) * c.n_kv_heads + h) * kRing * kD + col;
  const uint16_t* const nk = p.k.row(b, h, 0) + col;
  const uint16_t* const nv = p.v.row(b, h, 0) + col;
  uint4 k[kN], v[kN];
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    const int pos = i * kBlock + row0 + j * kRowsPass;
    if (pos >= start) {
      k[j] = ldg16(nk + int64_t(pos - start) * p.k.st);
      v[j] = ldg16(nv + int64_t(pos - start) * p.v.st);
    } else {  // plain loads: the CTA stores to the ring afterwards
      k[j] = *reinterpret_cast<const uint4*>(c.k_ring + ring + (pos % kRing) * kD);
      v[j] = *reinterpret_cast<const uint4*>(c.v_ring + ring + (pos % kRing) * kD);
    }
  }
  float2 m = make_float2(amax_of<kBf16, kN>(k), amax_of<kBf16, kN>(v));
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    m.x = fmaxf(m.x, __shfl_xor_sync(0xffffffffu, m.x, off));
    m.y = fmaxf(m.y, __shfl_xor_sync(0xffffffffu, m.y, off));
  }
  __syncthreads();  // red is free again
  if ((tid & 31) == 0) red[tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    m.x = fmaxf(m.x, red[w].x);
    m.y = fmaxf(m.y, red[w].y);
  }
  constexpr float kTop = kInt8 ? 127.f : 448.f;
  const float ks = fmaxf(__fdiv_rn(m.x, kTop), 0x1p-126f), vs = fmaxf(__fdiv_rn(m.y, kTop), 0x1p-126f);
  const bool kbad = !(m.x < INFINITY), vbad = !(m.y < INFINITY);
  const float ki = __frcp_rn(ks), vi = __frcp_rn(vs);
  const int page = c.page_table[int64_t(b) * c.max_blocks + i];
  if (page < 0 || page >= c.n_pages) {  // the block is not stored
    if (tid == 0) set_error(p.err, NSA_ERR_INVALID);
    return;
  }
  const int64_t rec = int64_t(page) * c.n_kv_heads + h;
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    const int64_t at = (rec * kBlock + row0 + j * kRowsPass) * kD + col;
    const uint2 z = make_uint2(0u, 0u);
    *reinterpret_cast<uint2*>(c.k_codes + at) = kbad ? z : codes8<kBf16, kInt8>(k[j], ki);
    *reinterpret_cast<uint2*>(c.v_codes + at) = vbad ? z : codes8<kBf16, kInt8>(v[j], vi);
  }
  if (tid == 0) c.scales[rec] = make_float2(kbad ? NAN : ks, vbad ? NAN : vs);
}

// A KV head's bit in unclean[b] says that its ring may hold a value that is not
// finite.  It is taken back where the ring begins anew, by the unit's CTA before
// that stores to it (with more than 32 heads two CTAs have a bit: it stays).
__device__ __forceinline__ int unclean_bit(int h) { return 1 << (h & 31); }
__device__ __forceinline__ void ring_anew(const Cache& c, const Span& span, int b, int h) {
  if (span.anew && c.n_kv_heads <= 32) atomicAnd(c.unclean + b, ~unclean_bit(h));
}

// Stores a unit's tokens of its last two blocks in the ring, as they came;
// threads `id` of `n` share the rows.
template <int kD, bool kBf16>
__device__ __forceinline__ void store_ring(const AppendParams& p, int b, int h, int start, int end, int id, int n) {
  constexpr int kVecs = kD / 8;
  const Cache& c = p.c;
  const int col = (id % kVecs) * 8;
  const int64_t ring = (int64_t(b) * c.n_kv_heads + h) * kRing * kD + col;
  const uint16_t* const nk = p.k.row(b, h, 0) + col;
  const uint16_t* const nv = p.v.row(b, h, 0) + col;
  for (int pos = max(start, (end / kBlock - 1) * kBlock) + id / kVecs; pos < end; pos += n / kVecs) {
    uint4 k = ldg16(nk + int64_t(pos - start) * p.k.st), v = ldg16(nv + int64_t(pos - start) * p.v.st);
    uint32_t* const w[8] = {&k.x, &k.y, &k.z, &k.w, &v.x, &v.y, &v.z, &v.w};
    uint32_t bad = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t mk = nonfinite_mask<kBf16>(*w[e]);
      *w[e] |= mk & 0x7fff7fffu;  // NaN
      bad |= mk;
    }
    if (bad) atomicOr(c.unclean + b, unclean_bit(h));
    *reinterpret_cast<uint4*>(c.k_ring + ring + (pos % kRing) * kD) = k;
    *reinterpret_cast<uint4*>(c.v_ring + ring + (pos % kRing) * kD) = v;
  }
}

// Grid (units, 1 + blocks that lie wholly in the new tokens).  y = 0
// takes a unit's first block, which may begin in the ring, and then stores
// the newest tokens there -- the same CTA, since the ring has room for two
// blocks only and the stores can overwrite what the first block reads.
template <int kD, bool kBf16, bool kInt8>
__global__ void __launch_bounds__(kThreads) kv8_append_kernel(const AppendParams p) {
  __shared__ Span span;
  __shared__ float2 red[kThreads / 32];
  grid_launch_dependents();
  grid_dependency_wait();
  const int tid = threadIdx.x, b = blockIdx.x / p.c.n_kv_heads, h = blockIdx.x % p.c.n_kv_heads;
  if (tid == 0) {
    span = take_span(p, b, p.c.n_kv_heads * gridDim.y);
    if (blockIdx.y == 0) ring_anew(p.c, span, b, h);
  }
  __syncthreads();
  if (!span.ok) return;
  const int start = span.start, end = span.end;
  for (int i = start / kBlock + blockIdx.y; i < end / kBlock; i += gridDim.y)
    quantize_block<kD, kBf16, kInt8>(p, b, h, i, start, tid, red);
  if (blockIdx.y == 0) {
    __syncthreads();  // every thread has read what it needs of the ring
    store_ring<kD, kBf16>(p, b, h, start, end, tid, kThreads);
  }
}

// The same for fewer new tokens than a block has, a smaller CTA a unit: most
// units only store a row or a few, so what counts is how many CTAs are resident
// at once; K and V of a block that is completed take turns in the registers (40
// of them: 6 CTAs an SM).  One token of 256 x 8 units: 6.2 us, 7.3 with the
// kernel above; 256 units that all complete a block: 2 us more than there (with
// 128 threads 5.7 us and 4 more, with 64 and the block read twice 12 and 30).
constexpr int kFewThreads = 256;
template <int kD, bool kBf16, bool kInt8>
__global__ void __launch_bounds__(kFewThreads) kv8_append_few_kernel(const AppendParams p) {
  constexpr int kVecs = kD / 8, kRowsPass = kFewThreads / kVecs, kN = kBlock / kRowsPass;
  constexpr float kTop = kInt8 ? 127.f : 448.f;
  __shared__ Span span;
  __shared__ float red[2][kFewThreads / 32];
  grid_launch_dependents();
  grid_dependency_wait();
  const Cache& c = p.c;
  const int tid = threadIdx.x, b = blockIdx.x / c.n_kv_heads, h = blockIdx.x % c.n_kv_heads;
  if (tid == 0) {
    span = take_span(p, b, c.n_kv_heads);
    ring_anew(c, span, b, h);
  }
  __syncthreads();
  if (!span.ok) return;
  const int start = span.start, end = span.end, i = start / kBlock;
  if (end / kBlock != i) {  // block i is completed
    const int page = c.page_table[int64_t(b) * c.max_blocks + i];
    if (page < 0 || page >= c.n_pages) {  // it is not stored
      if (tid == 0) set_error(p.err, NSA_ERR_INVALID);
    } else {
      const int64_t rec = int64_t(page) * c.n_kv_heads + h;
      const int col = (tid % kVecs) * 8, row0 = tid / kVecs;
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        const uint16_t* const ring = (t ? c.v_ring : c.k_ring) + int64_t(blockIdx.x) * kRing * kD + col;
        const Rows& rows = t ? p.v : p.k;
        const uint16_t* const fresh = rows.row(b, h, 0) + col;
        uint8_t* const codes = (t ? c.v_codes : c.k_codes) + rec * kBlock * kD + col;
        uint4 x[kN];
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          const int pos = i * kBlock + row0 + j * kRowsPass;
          x[j] = *reinterpret_cast<const uint4*>(pos >= start ? fresh + int64_t(pos - start) * rows.st
                                                              : ring + (pos % kRing) * kD);
        }
        float m = amax_of<kBf16, kN>(x);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
        if ((tid & 31) == 0) red[t][tid >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kFewThreads / 32; ++w) m = fmaxf(m, red[t][w]);
        const bool bad = !(m < INFINITY);
        const float scale = fmaxf(__fdiv_rn(m, kTop), 0x1p-126f), inv = __frcp_rn(scale);
#pragma unroll
        for (int j = 0; j < kN; ++j)
          *reinterpret_cast<uint2*>(codes + (row0 + j * kRowsPass) * kD) =
              bad ? make_uint2(0u, 0u) : codes8<kBf16, kInt8>(x[j], inv);
        if (tid == 0) reinterpret_cast<float*>(c.scales + rec)[t] = bad ? NAN : scale;
      }
    }
  }
  __syncthreads();  // every thread has read what it needs of the ring
  store_ring<kD, kBf16>(p, b, h, start, end, tid, kFewThreads);
}

// Sequences begin with pages that hold their first `lens` tokens already; one
// thread a sequence.
__global__ void __launch_bounds__(kThreads) kv8_adopt_kernel(const Cache c, const int64_t* lens, int* err) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int b = blockIdx.x * kThreads + threadIdx.x;
  if (b >= c.batch) return;
  const int64_t n = lens[b];
  if (n == -1) return;
  if (n < 0 || n > int64_t(c.max_blocks) * kBlock || n % kBlock) {
    set_error(err, NSA_ERR_INVALID);
    return;
  }
  c.lens[b] = n;
  c.ring_floor[b] = ring_state(n, n);  // the ring has nothing of them
  c.unclean[b] = 0;
}

// ---------------------------------------------------------------- read back
struct ReadParams {
  Cache c;
  int n_tokens;
  unsigned tiles;  // per unit
  const int64_t* starts;
  void *k_out, *v_out;
  int* err;
};

template <bool kInt8>
__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
  if constexpr (kInt8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int>(w << (24 - 8 * i)) >> 24);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t h;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(w >> (16 * i))));
      const float2 f = Elem<false>::unpack(h);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}

// kOut: 0 float32, 1 float16, 2 bfloat16
template <int kOut>
__device__ __forceinline__ void store8(void* out, int64_t at, const float (&x)[8]) {
  if constexpr (kOut == 0) {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
    o[0] = make_float4(x[0], x[1], x[2], x[3]);
    o[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    using E = Elem<kOut == 2>;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) =
        make_uint4(E::pack(x[0], x[1]), E::pack(x[2], x[3]), E::pack(x[4], x[5]), E::pack(x[6], x[7]));
  }
}

// One CTA a tile of kReadRows positions of a unit; a thread takes 8 elements of a
// row of K and of V, so that a warp's 16-byte stores fill whole sectors.  Bound
// by HBM (1 byte in, 2 out an element): all of a thread's loads are issued before
// its stores.  8 x 16,000 tokens, 8 heads of 128 to bf16: 124 us, 0.97 of the
// measured copy rate (16 elements a thread, each store half a sector a lane: 146;
// CTAs that take tiles in turn and look the next one's pages up ahead: 166).
constexpr int kReadRows = 64;
template <int kD, bool kBf16, bool kInt8, int kOut>
__global__ void __launch_bounds__(kThreads) kv8_read_kernel(const ReadParams p) {
  constexpr int kVecs = kD / 8, kRowsPass = kThreads / kVecs, kN = kReadRows / kRowsPass;
  grid_launch_dependents();
  grid_dependency_wait();
  const Cache& c = p.c;
  const int64_t unit = blockIdx.x / p.tiles, tile = blockIdx.x % p.tiles;
  const int b = static_cast<int>(unit / c.n_kv_heads), h = static_cast<int>(unit % c.n_kv_heads);
  const int64_t cap = int64_t(c.max_blocks) * kBlock;
  int64_t len = c.lens[b];
  if (len < 0 || len > cap) {
    if (threadIdx.x == 0) set_error(p.err, NSA_ERR_INVALID);
    len = 0;
  }
  const int64_t start = p.starts ? p.starts[b] : 0;
  const int64_t full = len / kBlock * kBlock;  // positions below are codes
  const int col = (threadIdx.x % kVecs) * 8, row0 = threadIdx.x / kVecs;
  uint2 kc[kN], vc[kN];
  float2 sc[kN];
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    const int64_t r = tile * kReadRows + row0 + j * kRowsPass, pos = start + r;
    kc[j] = vc[j] = make_uint2(0, 0);
    sc[j] = make_float2(0.f, 0.f);
    if (r < p.n_tokens && pos >= 0 && pos < full) {
      const int page = __ldg(c.page_table + int64_t(b) * c.max_blocks + pos / kBlock);
      if (page < 0 || page >= c.n_pages) {
        set_error(p.err, NSA_ERR_INVALID);
        sc[j] = make_float2(NAN, NAN);
      } else {
        const int64_t rec = int64_t(page) * c.n_kv_heads + h, at = (rec * kBlock + pos % kBlock) * kD + col;
        kc[j] = __ldg(reinterpret_cast<const uint2*>(c.k_codes + at));
        vc[j] = __ldg(reinterpret_cast<const uint2*>(c.v_codes + at));
        sc[j] = __ldg(c.scales + rec);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    const int64_t r = tile * kReadRows + row0 + j * kRowsPass, pos = start + r;
    if (r >= p.n_tokens) continue;
    const int64_t at = (unit * p.n_tokens + r) * kD + col;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float x[8];
      if (pos >= full && pos < len) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>((t ? c.v_ring : c.k_ring) +
                                                             (unit * kRing + pos % kRing) * kD + col));
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = Elem<kBf16>::unpack(ws[e]);
          x[2 * e] = f.x, x[2 * e + 1] = f.y;
        }
      } else {
        const uint2 w = t ? vc[j] : kc[j];
        const float s = t ? sc[j].y : sc[j].x;
        const uint32_t ws[2] = {w.x, w.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float y[4];
          decode4<kInt8>(ws[i], y);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[4 * i + e] = y[e] * s;
        }
      }
      store8<kOut>(t ? p.v_out : p.k_out, at, x);
    }
  }
}

template <int kD, bool kBf16, bool kInt8>
cudaError_t launch_append(const AppendParams& p, cudaStream_t stream) {
  const int64_t units = int64_t(p.c.batch) * p.c.n_kv_heads;
  if (p.n_tokens < kBlock) {  // at most one block is completed
    return launch_kernel(kv8_append_few_kernel<kD, kBf16, kInt8>, dim3(static_cast<unsigned>(units)), dim3(kFewThreads),
                         0, stream, p);
  }
  const int more = (p.n_tokens + kBlock - 1) / kBlock;  // blocks besides a unit's first
  int most = (1 << 30) / p.c.n_kv_heads - 2;  // three times a sequence's CTAs is an unsigned
  most = most < 65534 ? most : 65534;
  const dim3 grid(static_cast<unsigned>(units), 1 + static_cast<unsigned>(more < most ? more : most));
  return launch_kernel(kv8_append_kernel<kD, kBf16, kInt8>, grid, dim3(kThreads), 0, stream, p);
}
template <int kD, bool kBf16, bool kInt8>
cudaError_t launch_read(const ReadParams& p, int out_dtype, dim3 grid, cudaStream_t stream) {
  switch (out_dtype) {
    case 0: return launch_kernel(kv8_read_kernel<kD, kBf16, kInt8, 0>, grid, dim3(kThreads), 0, stream, p);
    case 1: return launch_kernel(kv8_read_kernel<kD, kBf16, kInt8, 1>, grid, dim3(kThreads), 0, stream, p);
    default: return launch_kernel(kv8_read_kernel<kD, kBf16, kInt8, 2>, grid, dim3(kThreads), 0, stream, p);
  }
}

// f<D, bf16, int8>(args...) for the descriptor's types
#define NSA_KV8_DISPATCH(c, f, ...)                                                                        \
  ((c)->head_dim == 128                                                                                    \
       ? ((c)->dtype == 2 ? ((c)->codes ? f<128, true, true>(__VA_ARGS__) : f<128, true, false>(__VA_ARGS__))    \
                          : ((c)->codes ? f<128, false, true>(__VA_ARGS__) : f<128, false, false>(__VA_ARGS__))) \
       : ((c)->dtype == 2 ? ((c)->codes ? f<64, true, true>(__VA_ARGS__) : f<64, true, false>(__VA_ARGS__))      \
                          : ((c)->codes ? f<64, false, true>(__VA_ARGS__) : f<64, false, false>(__VA_ARGS__))))

}  // namespace
}  // namespace kv8
}  // namespace nsa

using namespace nsa;

extern "C" int nsa_kv8_append(const nsa_kv8_cache* cache, const nsa_kv8_rows* new_k, const nsa_kv8_rows* new_v,
                              int64_t n_tokens, const int64_t* starts, const int64_t* counts, nsa_stream_t stream) {
  clear_error();
  kv8::AppendParams p{};
  int rc = kv8::check_cache(cache, p.c);
  if (rc) return rc;
  if (n_tokens < 0 || n_tokens > kv8::kMaxPos) return fail(NSA_ERR_INVALID, "n_tokens must be in [0, 2^30]");
  if (p.c.batch == 0) return NSA_OK;
  if (n_tokens > 0) {
    if ((rc = kv8::check_rows(new_k, "new_k", p.k))) return rc;
    if ((rc = kv8::check_rows(new_v, "new_v", p.v))) return rc;
  } else if (!starts) {
    return NSA_OK;  // nothing to write and no length to set
  }
  p.n_tokens = static_cast<int>(n_tokens);
  p.starts = starts;
  p.counts = counts;
  p.err = device_error_word();
  if (!p.err) return fail(NSA_ERR_CUDA, "device error word unavailable");
  cudaError_t e = NSA_KV8_DISPATCH(cache, kv8::launch_append, p, stream);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? NSA_OK : cuda_fail(e, "kv8_append_kernel launch");
}

extern "C" int nsa_kv8_adopt(const nsa_kv8_cache* cache, const int64_t* lens, nsa_stream_t stream) {
  clear_error();
  kv8::Cache c;
  const int rc = kv8::check_cache(cache, c);
  if (rc) return rc;
  if (c.batch == 0) return NSA_OK;
  if (!lens) return fail(NSA_ERR_INVALID, "lens is NULL");
  int* const err = device_error_word();
  if (!err) return fail(NSA_ERR_CUDA, "device error word unavailable");
  cudaError_t e = launch_kernel(kv8::kv8_adopt_kernel, dim3((c.batch + kv8::kThreads - 1) / kv8::kThreads), dim3(kv8::kThreads),
                                0, stream, c, lens, err);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? NSA_OK : cuda_fail(e, "kv8_adopt_kernel launch");
}

extern "C" int nsa_kv8_read(const nsa_kv8_cache* cache, int64_t n_tokens, const int64_t* starts, void* k_out,
                            void* v_out, int out_dtype, nsa_stream_t stream) {
  clear_error();
  kv8::ReadParams p{};
  int rc = kv8::check_cache(cache, p.c);
  if (rc) return rc;
  if (n_tokens < 0 || n_tokens > kv8::kMaxPos) return fail(NSA_ERR_INVALID, "n_tokens must be in [0, 2^30]");
  if (out_dtype < 0 || out_dtype > 2) return fail(NSA_ERR_UNSUPPORTED, "out_dtype must be 0, 1 or 2");
  if (p.c.batch == 0 || n_tokens == 0) return NSA_OK;
  if (!k_out || !v_out) return fail(NSA_ERR_INVALID, "null pointer");
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(NSA_ERR_ALIGN, "outputs must be 16-byte aligned");
  const int64_t units = int64_t(p.c.batch) * p.c.n_kv_heads;
  p.n_tokens = static_cast<int>(n_tokens);
  p.starts = starts;
  p.k_out = k_out;
  p.v_out = v_out;
  p.err = device_error_word();
  if (!p.err) return fail(NSA_ERR_CUDA, "device error word unavailable");
  p.tiles = static_cast<unsigned>((n_tokens + kv8::kReadRows - 1) / kv8::kReadRows);
  if (units * p.tiles > 0x7fffffff) return fail(NSA_ERR_UNSUPPORTED, "too many tokens for one read");
  const dim3 grid(static_cast<unsigned>(units * p.tiles));
  cudaError_t e = NSA_KV8_DISPATCH(cache, kv8::launch_read, p, out_dtype, grid, stream);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? NSA_OK : cuda_fail(e, "kv8_read_kernel launch");
}
