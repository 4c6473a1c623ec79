// Attention over the 8-bit paged cache, for the last 1 to 64 tokens of every
// sequence (decode, verification of drafts).
//
//   o[n] = sum_p softmax_p(scale * q[n] . k[p]) v[p],  k[p] = ks(block of p) * kc[p], v likewise
//
// The scales leave the products: s = ks * (q . kc), o = sum over blocks of
// vs * (P . vc).  The codes become fp16 exactly (e4m3 and int8 both fit), so the
// products run on mma.sync m16n8k16 with fp16 operands and fp32 sums.  Queries
// enter as fp16 after a power of two per row has brought their largest element
// into [2^15, 2^16): exact for fp16, and for bf16 but for elements 2^-32 below
// the row's largest, which keep an absolute error of 2^-40 of it.
//
// Bound by HBM for up to 8 query rows a KV head, which take 16 FLOP a byte (4 x
// 163,840 tokens, 64 / 8 heads of 128: 211 us, 0.98 of the measured copy rate); by
// the instructions around the products for more (32 rows: 0.26).  tcgen05 would
// want the codes as fp16 in shared memory first and tiles of 64 or 128 rows; here
// the conversion happens in registers on the way from ldmatrix to the mma.
// Short calls are bound by the way from the lengths to the first load (3 us from
// the launch to the page number, 2 more to its keys) and by one step's
// latency (2.6 us); B = 1, L = 512 takes 10 us.
//
// Work is split evenly over independent workers (warps) by steps: a step is a
// block of 64 tokens, or 32 tokens of a sequence's incomplete block in the
// ring.  The lengths live on the device, so every CTA computes the split itself
// (one scan over the batch).  A worker issues its own TMA loads -- the next K as
// soon as the scores are done, the next V as soon as the sums are -- and keeps
// scores, P and accumulators in registers, so no warp waits for another until
// its steps are done.  A worker's consecutive steps form pieces of units
// (sequence, KV head, row tile).  Units cut between workers are merged by the
// CTA at its end, and those cut between CTAs by the last of them to finish.
#include <cstddef>

#include "kv8.cuh"

namespace nsa {
namespace kv8 {
namespace {

constexpr int kShare = 6;   // steps of a CTA at least, where there are more CTAs than units
constexpr int kMerge = 16;  // steps that take a CTA as long as a merge across CTAs
constexpr int kLensCached = 512;  // sequence lengths kept in shared memory
constexpr float kLog2e = 1.4426950408889634f;

struct AttendParams {
  Cache c;
  Rows q, o;
  int group, n_tokens, rows, row_tiles;  // rows = n_tokens * group of a KV head
  uint32_t group_inv;                    // ceil(2^32 / group)
  float units_inv;                       // 1 / (KV heads * row_tiles)
  const int64_t* counts;
  int window, sink;  // window < 0: all positions
  float scale_log2;
  int* tickets;     // [CTAs]
  float* partials;  // [workers][2] pieces, then [CTAs][2]: maximum and sum of every row, then kD sums a row
  int* err;
};

// n / group; exact for n < 2^16, group <= 2^10 (the error of group_inv adds
// less than n / 2^32 to a quotient that is at least 1 / group below the next).
__device__ __forceinline__ int token_of(const AttendParams& p, int n) {
  return p.group == 1 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), p.group_inv));
}

constexpr int kRingTok = 32;  // tokens of a ring step

template <int kD>
struct Geo {
  static constexpr uint32_t kHalf = kBlock * kD;  // bytes of K, and of V, of a step (ring: 32 tokens of 2 bytes)
  static constexpr uint32_t kRegions = kD / 64;   // 128-byte column parts of a ring step
  static constexpr uint32_t kRegion = kRingTok * 128;
};

// One sequence as the kernel sees it.
struct Seq {
  int len, cnt;                // tokens; query tokens (rows of later ones are 0)
  int full;                    // complete blocks
  int sink_blocks, win_block;  // blocks read: [0, sink_blocks), [win_block, full)
  int steps;                   // at least 1
  bool empty;                  // nothing to see: its one step writes zeros
};

__device__ __forceinline__ Seq make_seq(const AttendParams& p, int len, int cnt) {
  Seq s;
  s.len = len;
  s.cnt = cnt;
  s.full = len / kBlock;
  s.sink_blocks = 0;
  s.win_block = 0;
  if (p.window >= 0) {
    s.sink_blocks = min((p.sink + kBlock - 1) / kBlock, s.full);
    s.win_block = min(max(max(len - cnt + 1 - p.window, 0) / kBlock, s.sink_blocks), s.full);
  }
  s.steps = s.sink_blocks + s.full - s.win_block + (len % kBlock + kRingTok - 1) / kRingTok;
  s.empty = cnt == 0 || s.steps == 0;
  if (s.empty) s.steps = 1;
  return s;
}

// A sequence's length and query count, checked: an invalid one reads as an
// empty sequence.
__device__ __forceinline__ int2 load_len(const AttendParams& p, int b) {
  const int64_t len = p.c.lens[b];
  const int64_t cnt = p.counts ? p.counts[b] : p.n_tokens;
  if (len < 0 || len > int64_t(p.c.max_blocks) * kBlock || cnt < 0 || cnt > p.n_tokens) {
    set_error(p.err, NSA_ERR_INVALID);
    return make_int2(0, 0);
  }
  return make_int2(static_cast<int>(len), static_cast<int>(cnt));
}

// What a worker has to know of a step.
struct Step {
  int b, sub;    // sequence; KV head * row_tiles + row tile
  int len, cnt;  // of the sequence
  int pos0;      // position of its first token
  int flags;     // kFirst..., and from bit 16 on the tokens of a ring step
  int step, steps;  // which of its unit's
  float ks, vs;  // scales
  int row;       // of the tensor map
};
enum : int {
  kFirst = 1,   // of the worker's piece
  kLast = 2,
  kBegin = 4,   // of the unit
  kEnd = 8,
  kRingStep = 16,
  kEmpty = 32,
  kMasked = 64,  // some row does not see some of its tokens
  kUnclean = 128  // the ring may hold values that are not finite
};

// A worker's part of a cut unit.
struct Part {
  int unit_begin;  // the unit's first step
  float* data;
  int b, sub, cnt, steps;
  int flags;  // 0: none; else kFirst and whether it holds the unit's begin / end
};

// One CTA per SM.  12 warps of 168 registers where the accumulators leave room
// (up to 8 query rows of 128 dimensions, 16 of 64), else 8 of 255.  Spilled
// registers are dear here: with this much shared memory they miss the L1.
template <int kD, int kNT>
struct Shape {
  static constexpr int kWarps = kNT * kD <= 128 ? 12 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kRows = 8 * kNT;  // of a unit
  static constexpr int kQStride = kD * 2 + 32;  // bytes: rows 8 banks apart
  static constexpr int kTok = 32;  // tokens of a round of scores, softmax and sums
};

template <int kD, int kNT>
struct Smem {
  using H = Shape<kD, kNT>;
  uint8_t stage[H::kWarps][2 * Geo<kD>::kHalf];  // K, V; 1024-aligned: TMA destinations
  uint8_t q[H::kWarps][H::kRows][H::kQStride];
  Part part[H::kWarps][2];
  int2 lens[kLensCached];
  int2 scan[H::kWarps];  // steps and the longest unit of each warp's sequences
  int before[H::kThreads];  // steps before a thread's sequences
  int last[2];  // whether this CTA was the last of its first / last cut unit
  uint64_t k_full[H::kWarps], v_full[H::kWarps];
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool kBf16>
__device__ __forceinline__ void mma_elem(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    mma_bf16(d, a0, a1, a2, a3, b0, b1);
  else
    mma_16816(d, a0, a1, a2, a3, b0, b1);
}

// D = A * B (mma_16816 without a sum to go on from).
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// Two 16 x 16 matrices of bytes, transposed: lane (g, t) gets of each the rows
// 4t .. 4t + 3 of columns g and g + 8.
__device__ __forceinline__ void ldmatrix_b8_trans(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2,
                                                  uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}

// Four codes to two fp16 pairs.  int8: the byte, biased by 128, is the low part of an
// fp16 number in [1024, 2048), from which 1152 is taken again (exact).
template <bool kInt8>
__device__ __forceinline__ void to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kInt8) {
    const uint32_t x = w ^ 0x80808080u, magic = 0x64646464u;
    const uint32_t a = __byte_perm(x, magic, 0x4140);
    const uint32_t b = __byte_perm(x, magic, 0x4342);
    const __half2 bias = __float2half2_rn(1152.f);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&a), bias);
    const __half2 z = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
    lo = *reinterpret_cast<const uint32_t*>(&y);
    hi = *reinterpret_cast<const uint32_t*>(&z);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

__device__ __forceinline__ void lds8(uint32_t addr, uint32_t& lo, uint32_t& hi) {
  // (memory: it may read what plain stores have written)
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(lo), "=r"(hi) : "r"(addr) : "memory");
}
// A pair of fp16 numbers of 8 significant bits times 2^-15 as bf16 (exact; as
// they are, the products with bf16 tokens would have no room).  volatile, so that
// the conversions of all query fragments stay on the ring's path instead of
// being kept in registers.
__device__ __forceinline__ uint32_t half_to_bf16(uint32_t x) {
  uint32_t y;
  asm volatile(
      "{\n\t.reg .b16 l, h;\n\t.reg .f32 a, b;\n\tmov.b32 {l, h}, %1;\n\tcvt.f32.f16 a, l;\n\tcvt.f32.f16 b, h;\n\t"
      "mul.f32 a, a, 0f38000000;\n\tmul.f32 b, b, 0f38000000;\n\t"
      "cvt.rn.bf16x2.f32 %0, b, a;\n\t}"
      : "=r"(y)
      : "r"(x));
  return y;
}

// Whether a row with position limit `lim` sees `pos`.
__device__ __forceinline__ bool sees(const AttendParams& p, int pos, int lim) {
  return pos < lim && (p.window < 0 || pos < p.sink || pos >= lim - p.window);
}

// A pair of float32 numbers as 16-bit ones and what that rounding left.
template <bool kBf16>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = Elem<kBf16>::pack(x, y);
  const float2 back = Elem<kBf16>::unpack(hi);
  lo = Elem<kBf16>::pack(x - back.x, y - back.y);
}

// The even split of `total` > 0 steps over at most `most` takers: the first
// `rem` of n take one step more than the others, and takers from n on nothing.
struct Split {
  uint32_t total, n, each, rem;
  __device__ __forceinline__ Split(uint32_t total_, uint32_t most) : total(total_), n(min(most, total_)) {
    each = total / n;
    rem = total - each * n;
  }
  __device__ __forceinline__ uint32_t begin(uint32_t g) const { return g < n ? g * each + min(g, rem) : total; }
  __device__ __forceinline__ uint32_t owner(uint32_t x) const {
    const uint32_t wide = rem * (each + 1);
    return x < wide ? x / (each + 1) : rem + (x - wide) / each;
  }
};

template <bool kCg, class T>
__device__ __forceinline__ T load(const T* p) {
  if constexpr (kCg) return __ldcg(p);
  return *p;
}

// Row `row` of pieces that cover a unit (or a part of it): their sums under a
// common maximum.  A lane holds one piece's maximum and sum at a time, then
// kD / 32 columns.  ptr(i): the data of piece i < n, with kCg written by other
// CTAs (read past the L1).
template <int kD, int kRows, bool kCg, class Ptr>
__device__ __forceinline__ void merge_row(int n, int row, int lane, Ptr ptr, float& M, float& L, float (&a)[kD / 32]) {
  constexpr int kCols = kD / 32;
  M = -INFINITY;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, load<kCg>(reinterpret_cast<const float2*>(ptr(i)) + row).x);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
  const float ref = M == -INFINITY ? 0.f : M;
  L = 0.f;
#pragma unroll
  for (int k = 0; k < kCols; ++k) a[k] = 0.f;
  for (int i0 = 0; i0 < n; i0 += 32) {
    float w = 0.f;
    if (i0 + lane < n) {
      const float2 ml = load<kCg>(reinterpret_cast<const float2*>(ptr(i0 + lane)) + row);
      w = fast_exp2(ml.x - ref);
      L += ml.x == -INFINITY ? ml.y : w * ml.y;  // (a row of NaN scores has no maximum; its sum is NaN)
    }
    const int cnt = min(32, n - i0);
#pragma unroll 4
    for (int j = 0; j < cnt; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const float* src = ptr(i0 + j) + 2 * kRows + row * kD + lane * kCols;
      if constexpr (kCols == 4) {
        const float4 x = load<kCg>(reinterpret_cast<const float4*>(src));
        a[0] += wj * x.x, a[1] += wj * x.y, a[2] += wj * x.z, a[3] += wj * x.w;
      } else {
        const float2 x = load<kCg>(reinterpret_cast<const float2*>(src));
        a[0] += wj * x.x, a[1] += wj * x.y;
      }
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
}

template <int kD, int kNT, bool kBf16, bool kInt8>
__global__ void __launch_bounds__(Shape<kD, kNT>::kThreads, 1)
    kv8_attend_kernel(const __grid_constant__ CUtensorMap tm_kc, const __grid_constant__ CUtensorMap tm_vc,
                      const __grid_constant__ CUtensorMap tm_kr, const __grid_constant__ CUtensorMap tm_vr,
                      const AttendParams p) {
  using G = Geo<kD>;
  using H = Shape<kD, kNT>;
  using S = Smem<kD, kNT>;
  constexpr int kRows = H::kRows;
  constexpr int kChunks = kD / 16;              // 16-wide steps of the head dimension
  constexpr int kTC = H::kTok / 16;             // 16-token parts of a round
  constexpr int kRounds = kBlock / H::kTok;
  constexpr int kRC = kTC < kRingTok / 16 ? kTC : kRingTok / 16;  // of a round of a ring step
  constexpr int kPiece = kRows * (2 + kD);      // floats of a partial result
  constexpr int kKUnroll = 2;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  grid_launch_dependents();
  if (smem_u32(smem_raw) & 1023u) {
    if (threadIdx.x == 0) set_error(p.err, NSA_ERR_ALIGN);
    return;
  }
  S& sm = *reinterpret_cast<S*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (tid < H::kWarps) {
    mbar_init(smem_u32(&sm.k_full[tid]), 1);
    mbar_init(smem_u32(&sm.v_full[tid]), 1);
    fence_barrier_init();
  }
  if (tid < 2 * H::kWarps) sm.part[tid >> 1][tid & 1].flags = 0;
  if (tid == H::kThreads - 1) {
    prefetch_tmap(&tm_kc);
    prefetch_tmap(&tm_vc);
    prefetch_tmap(&tm_kr);
    prefetch_tmap(&tm_vr);
  }
  grid_dependency_wait();

  // ---- the split: steps before each thread's run of sequences
  const int batch = p.c.batch, per = (batch + H::kThreads - 1) / H::kThreads;
  const int units = p.c.n_kv_heads * p.row_tiles;  // of a sequence
  int mine = 0, longest = 0;  // steps of this thread's sequences, of one unit
  for (int b = tid * per; b < min(batch, (tid + 1) * per); ++b) {
    const int2 l = load_len(p, b);
    if (b < kLensCached) sm.lens[b] = l;
    const int steps = make_seq(p, l.x, l.y).steps;
    mine += steps;
    longest = max(longest, steps);
  }
  int before = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, before, off);
    if (lane >= off) before += y;
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (lane == 31) sm.scan[warp] = make_int2(before, longest);
  __syncthreads();
  const int2 of_warp = lane < H::kWarps ? sm.scan[lane] : make_int2(0, 0);
  const int sum = __reduce_add_sync(0xffffffffu, of_warp.x);
  const int prior = __reduce_add_sync(0xffffffffu, lane < warp ? of_warp.x : 0);
  longest = __reduce_max_sync(0xffffffffu, of_warp.y);
  if (__umulhi(sum, units) != 0 || static_cast<int>(static_cast<uint32_t>(sum) * units) < 0) {  // (16 TB of codes)
    if (tid == 0) set_error(p.err, NSA_ERR_INVALID);
    return;
  }
  sm.before[tid] = before + prior - mine;
  __syncthreads();
  // a CTA for every kShare steps, or for every unit
  const uint32_t total = static_cast<uint32_t>(sum) * units;
  const Split split(total, min(gridDim.x, max((total + kShare - 1) / kShare, static_cast<uint32_t>(batch * units))));
  if (blockIdx.x >= split.n) return;
  // A CTA's range ends at a unit's border where that costs less than a merge
  // across CTAs, about kMerge steps of a CTA's time: where the unit there has at
  // most twice as many (a border moves by half of it at most), and everywhere
  // where the CTA with most units has few steps above the average.  (B = 16, L =
  // 4096, 8 KV heads: 37.5 us with cut units, 31 with whole ones; B = 1: 18 and 26.)
  // (a quotient one too low or high only shifts that choice, the same for all)
  const int whole_each = static_cast<int>(__fdividef(static_cast<float>(split.each + kMerge), static_cast<float>(longest)));
  const int whole = batch * units <= static_cast<int>(split.n) * whole_each ? longest : 2 * kMerge;
  // Which sequence holds step x?  Asked for the CTA's two borders, by the halves
  // of every warp, and again for the warp's own first step where that is not in
  // the first border's sequence.
  int x = split.begin(blockIdx.x + (lane >> 4));
  const int threads = (batch + per - 1) / per;
  int cur_b = 0, cur_rel = 0;  // a sequence, and its first step from the worker's first
  int x0 = 0, n_steps = 0;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    const int ask = pass == 0 && x == static_cast<int>(total) ? 0 : x;
    // ask / units: a quotient in float32, what it left over divided again, and one step at most to go
    int at = __float2int_rz(__int2float_rz(ask) * p.units_inv);
    at += __float2int_rn(__int2float_rn(ask - at * units) * p.units_inv);
    at -= at * units > ask;
    at += (at + 1) * units <= ask;
    int n = 0;
#pragma unroll 1
    for (int i = lane & 15; i < threads; i += 16) n += sm.before[i] <= at;
    n = __reduce_add_sync(lane < 16 ? 0xffffu : 0xffff0000u, n) - 1;  // the last run that begins at it or before
    cur_b = n * per;
    int begin = sm.before[n], steps;
    for (;;) {
      const int2 l = cur_b < kLensCached ? sm.lens[cur_b] : load_len(p, cur_b);
      steps = make_seq(p, l.x, l.y).steps;
      if (at < begin + steps) break;
      begin += steps;
      ++cur_b;
    }
    begin *= units;
    if (pass == 0) {
      if (ask > 0 && steps <= whole) {
        const int in = (x - begin) % steps;
        x += 2 * in < steps ? -in : steps - in;
      }
      __syncwarp();
      const int lo = __shfl_sync(0xffffffffu, x, 0), cta_steps = __shfl_sync(0xffffffffu, x, 16) - lo;
      if (cta_steps == 0) return;  // the whole CTA
      // workers with steps are the first ones: their parts follow one another
      const int each = cta_steps / H::kWarps, rem = cta_steps - each * H::kWarps;
      x0 = x = lo + warp * each + min(warp, rem);
      n_steps = each + (warp < rem);
      if (n_steps == 0) x = lo;  // (asks for anything)
      cur_b = __shfl_sync(0xffffffffu, cur_b, 0);
      begin = __shfl_sync(0xffffffffu, begin, 0);
      steps = __shfl_sync(0xffffffffu, steps, 0);
      cur_rel = begin - x;
      if (x < begin + steps * units) break;
    } else {
      cur_rel = begin - x;
    }
  }
  const uint32_t worker = blockIdx.x * H::kWarps + warp;

  // ---- issuing: lane i knows step batch0 + i
  int batch0 = -32;
  Step ahead{};
  auto head_of = [&](int sub) { return p.row_tiles == 1 ? sub : sub / p.row_tiles; };
  auto limit_at = [&](int len, int cnt, int n) {
    return max(len - cnt + 1 + min(token_of(p, min(n, p.rows - 1)), cnt - 1), 0);
  };
  auto fetch = [&](int k0) {
    batch0 = k0;
    const int k = k0 + lane, k_end = min(k0 + 32, n_steps);
    bool found = k >= n_steps;
    Seq s;
    int step = 0, sub = 0, b = 0;
    for (;;) {
      const int2 l = cur_b < kLensCached ? sm.lens[cur_b] : load_len(p, cur_b);
      const Seq c = make_seq(p, l.x, l.y);
      const int end = cur_rel + c.steps * units;
      if (!found && k < end) {
        const uint32_t off = static_cast<uint32_t>(k - cur_rel);
        sub = off / static_cast<uint32_t>(c.steps);
        step = off - sub * c.steps;
        b = cur_b;
        s = c;
        found = true;
      }
      if (k_end <= end) break;
      ++cur_b;
      cur_rel = end;
    }
    if (k >= n_steps) return;
    const int h = head_of(sub), n0 = (sub - h * p.row_tiles) * kRows;
    ahead.b = b;
    ahead.sub = sub;
    ahead.len = s.len;
    ahead.cnt = s.cnt;
    ahead.step = step;
    ahead.steps = s.steps;
    ahead.pos0 = 0;
    ahead.ks = ahead.vs = 1.f;
    int flags = (step == 0 ? kBegin | kFirst : 0) | (step == s.steps - 1 ? kEnd | kLast : 0);
    flags |= (k == 0 ? kFirst : 0) | (k == n_steps - 1 ? kLast : 0);
    const int blocks = s.sink_blocks + s.full - s.win_block;
    if (s.empty) {
      flags |= kEmpty;
    } else if (step < blocks) {
      const int block = step < s.sink_blocks ? step : s.win_block + step - s.sink_blocks;
      int page = __ldg(p.c.page_table + int64_t(b) * p.c.max_blocks + block);
      float2 sc = make_float2(NAN, NAN);
      if (page >= 0 && page < p.c.n_pages) {
        sc = __ldg(p.c.scales + int64_t(page) * p.c.n_kv_heads + h);
      } else {
        set_error(p.err, NSA_ERR_INVALID);
        page = 0;
      }
      ahead.ks = sc.x;
      ahead.vs = sc.y;
      ahead.pos0 = block * kBlock;
      ahead.row = (page * p.c.n_kv_heads + h) * kBlock;
      const int lo = limit_at(s.len, s.cnt, n0), hi = limit_at(s.len, s.cnt, n0 + kRows - 1);
      if (ahead.pos0 + kBlock > lo || (p.window >= 0 && ahead.pos0 < hi - p.window && ahead.pos0 + kBlock > p.sink))
        flags |= kMasked;
    } else {
      ahead.pos0 = s.full * kBlock + (step - blocks) * kRingTok;
      ahead.row = (b * p.c.n_kv_heads + h) * kRing + ahead.pos0 % kRing;
      flags |= kRingStep | kMasked | (p.c.unclean[b] >> (h & 31) & 1 ? kUnclean : 0) | (min(kRingTok, s.len - ahead.pos0) << 16);
    }
    ahead.flags = flags;
  };
  // Stages K (and with it the queries of a new piece) or V of step k; called for
  // k = 0, 1, ... in turn, K before V.
  int next_flags = 0, next_row = 0;
  auto issue = [&](int k, bool v) {
    if (k >= n_steps) return;
    const uint32_t fb = smem_u32(v ? &sm.v_full[warp] : &sm.k_full[warp]);
    uint32_t bytes = 0;
    if (!v) {
      if (k >= batch0 + 32) fetch(k);
      next_flags = __shfl_sync(0xffffffffu, ahead.flags, k - batch0);
      next_row = __shfl_sync(0xffffffffu, ahead.row, k - batch0);
      if ((next_flags & (kFirst | kEmpty)) == kFirst) {  // a query row a lane
        const int b = __shfl_sync(0xffffffffu, ahead.b, k - batch0), sub = __shfl_sync(0xffffffffu, ahead.sub, k - batch0);
        const int h = head_of(sub), n0 = (sub - h * p.row_tiles) * kRows, n_rows = min(kRows, p.rows - n0);
        fence_proxy_async_smem();  // the last piece's fragments were plain stores
        __syncwarp();
        if (lane < n_rows) {
          const int n = n0 + lane, tok = token_of(p, n);
          bulk_load(smem_u32(sm.q[warp][lane]), p.q.row(b, h * p.group + n - tok * p.group, tok), kD * 2, fb);
        }
        bytes = n_rows * kD * 2;
      }
    }
    const uint32_t dst = smem_u32(sm.stage[warp]) + (v ? G::kHalf : 0);
    if (lane == 0) {
      if (next_flags & kRingStep) {
        const int boxes = ((next_flags >> 16) + 7) / 8;  // of 8 slots, those that hold tokens
        mbar_arrive_expect_tx(fb, bytes + boxes * 16 * kD);
        for (int r = 0; r < boxes; ++r)
          for (uint32_t c = 0; c < G::kRegions; ++c)
            tma_load_2d(dst + c * G::kRegion + r * 1024, v ? &tm_vr : &tm_kr, fb, c * 64, next_row + 8 * r);
      } else if (!(next_flags & kEmpty)) {
        mbar_arrive_expect_tx(fb, bytes + G::kHalf);
        tma_load_2d(dst, v ? &tm_vc : &tm_kc, fb, 0, next_row);
      } else {
        mbar_arrive(fb);
      }
    }
    __syncwarp();
  };

  // ---- the worker's steps.  After a wait that ran out (the error word is
  // set) a warp waits no more, so that it still reaches the CTA's barriers.
  float qscale[kNT][2];  // of rows 8nt + 2t + (0, 1): the row's power of two (times 2^14), sm_scale and log2(e)
  float m[kNT][2], l[kNT][2];
  float acc[kNT][kChunks][4];  // dims 16c + g (0, 1) and 16c + g + 8 (2, 3), rows 2t (0, 2) and 2t + 1 (1, 3)
  bool begins = false;         // the piece holds its unit's first step
  bool aborted = false;
  const uint32_t q_at = smem_u32(&sm.q[warp][g][8 * t]);
  // 16 tokens of K are rows 0..15 of a product.  Row r < 8 is token r, row 8 +
  // j token 8 + (j ^ 4), so that the byte transposition of V, whose rows 4a +
  // (0..3) are then rows 2a, 2a + 1, 8 + 2a and 9 + 2a of the product, reads
  // eight different 16-byte columns of the swizzle at a time, as K does.
  const int k_hi = (lane >> 3) & 1, k_row = 8 * k_hi + ((lane & 7) ^ (k_hi << 2));
  const int v_a = (lane >> 2) & 3, v_j = lane & 3, v_row = v_j < 2 ? 2 * v_a + v_j : 8 + ((2 * v_a + v_j - 2) ^ 4);
  const uint32_t k_off = k_row * kD + (((lane >> 4) ^ (kD == 128 ? (k_row & 7) : ((k_row >> 1) & 3))) << 4);
  const uint32_t v_off = v_row * kD + (((lane >> 4) ^ (kD == 128 ? (v_row & 7) : ((v_row >> 1) & 3))) << 4);
  Step s{};
  s.flags = kEmpty;
  for (int k = -1; k < n_steps; ++k) {  // (step -1 only issues the first)
    if (k >= 0) {
      const int from = k - batch0;
      s.flags = next_flags;
      s.pos0 = __shfl_sync(0xffffffffu, ahead.pos0, from);
      s.step = __shfl_sync(0xffffffffu, ahead.step, from);
      s.steps = __shfl_sync(0xffffffffu, ahead.steps, from);
      s.ks = __shfl_sync(0xffffffffu, ahead.ks, from);
      s.vs = __shfl_sync(0xffffffffu, ahead.vs, from);
      if (s.flags & kFirst) {
        s.b = __shfl_sync(0xffffffffu, ahead.b, from);
        s.sub = __shfl_sync(0xffffffffu, ahead.sub, from);
        s.len = __shfl_sync(0xffffffffu, ahead.len, from);
        s.cnt = __shfl_sync(0xffffffffu, ahead.cnt, from);
      }
    }
    const bool ring = s.flags & kRingStep, empty = s.flags & kEmpty;
    if (k >= 0 && !aborted && !mbar_wait(smem_u32(&sm.k_full[warp]), k & 1, p.err)) aborted = true;
    if (s.flags & kFirst) {
      begins = s.flags & kBegin;
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) m[nt][e] = -INFINITY, l[nt][e] = 0.f;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[nt][c][e] = 0.f;
      }
      if (!empty) {
        // queries: fp16 fragments, k index permuted as the codes' ldmatrix gives it
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          uint2* const row = reinterpret_cast<uint2*>(&sm.q[warp][8 * nt + g][8 * t]);  // (every fourth of it)
          float top = 0.f;  // (rows that do not exist hold anything; nothing of them is stored)
#pragma unroll 2
          for (int c = 0; c < kChunks; ++c) {
            const uint2 x = row[4 * c];
            const float2 a = Elem<kBf16>::unpack(x.x), b = Elem<kBf16>::unpack(x.y);
            top = fmaxf(top, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          // a power of two from the exponent field; rows with infinities as they are
          int ex = static_cast<int>(__float_as_uint(top) >> 23);
          ex = ex == 255 ? 142 : max(ex, 15);
          const float f = __uint_as_float(static_cast<uint32_t>(269 - ex) << 23);
          const float back = __uint_as_float(static_cast<uint32_t>(ex - 1) << 23) * p.scale_log2;  // 2^14 / f
#pragma unroll 2
          for (int c = 0; c < kChunks; ++c) {
            const uint2 x = row[4 * c];
            const float2 a = Elem<kBf16>::unpack(x.x), b = Elem<kBf16>::unpack(x.y);
            row[4 * c] = make_uint2(pack_half2(a.x * f, a.y * f), pack_half2(b.x * f, b.y * f));
          }
          qscale[nt][0] = __shfl_sync(0xffffffffu, back, 8 * t);      // from a lane of row 2t
          qscale[nt][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);  // and of 2t + 1
        }
      }
    }
    auto q_frag = [&](int nt, int c, uint32_t& b0, uint32_t& b1) {  // (a lane reads what it wrote)
      lds8(q_at + nt * 8 * H::kQStride + 32 * c, b0, b1);
    };
    const uint32_t kb = smem_u32(sm.stage[warp]), vb = kb + G::kHalf;
    const int n_tok = s.flags >> 16;  // of a ring step
    const int rounds = ring ? (n_tok + H::kTok - 1) / H::kTok : kRounds;

#pragma unroll 1
    for (int round = 0; round < rounds; ++round) {
      float sc[kTC][kNT][4];
#pragma unroll
      for (int i = 0; i < kTC; ++i)
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[i][nt][e] = 0.f;
      if (!empty) {
        // ---- scores, S^T: rows g (0, 1) and g + 8 (2, 3) of 16 tokens; query rows 2t, 2t + 1
        if (!ring) {
          const uint32_t ka = kb + k_off + round * H::kTok * kD;
#pragma unroll kKUnroll
          for (int c = 0; c < kChunks; c += 2) {
            const uint32_t kc = ka ^ (c << 4);  // (its column is below the row's 128 or 64 bytes)
#pragma unroll
            for (int i = 0; i < kTC; ++i) {
              uint32_t r[4];
              ldmatrix_x4(kc + 16 * i * kD, r[0], r[1], r[2], r[3]);
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                uint32_t a0, a1, a2, a3;
                to_half<kInt8>(r[2 * j], a0, a2);
                to_half<kInt8>(r[2 * j + 1], a1, a3);
#pragma unroll
                for (int nt = 0; nt < kNT; ++nt) {
                  uint32_t b0, b1;
                  q_frag(nt, c + j, b0, b1);
                  mma_16816(sc[i][nt], a0, a1, a2, a3, b0, b1);
                }
              }
            }
          }
        } else {
#pragma unroll kKUnroll
          for (int c = 0; c < kChunks; ++c) {
            uint32_t b0[kNT], b1[kNT];
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) {
              q_frag(nt, c, b0[nt], b1[nt]);
              if constexpr (kBf16) b0[nt] = half_to_bf16(b0[nt]), b1[nt] = half_to_bf16(b1[nt]);
            }
#pragma unroll
            for (int i = 0; i < kRC; ++i) {
              // row & 7 == g for both of this lane's rows (those behind the tokens hold anything: masked below)
              const uint32_t at = kb + (c >> 2) * G::kRegion + (round * H::kTok + 16 * i + g) * 128 +
                                  ((((c & 3) * 2 + (t >> 1)) ^ g) << 4) + (t & 1) * 8;
              uint32_t a0, a1, a2, a3;
              lds8(at, a0, a2);
              lds8(at + 8 * 128, a1, a3);
#pragma unroll
              for (int nt = 0; nt < kNT; ++nt) mma_elem<kBf16>(sc[i][nt], a0, a1, a2, a3, b0[nt], b1[nt]);
            }
          }
        }
      }
      if (round == rounds - 1) {
        __syncwarp();
        issue(k + 1, false);
      }
      if (!empty) {
        const float q_unit = kBf16 && ring ? 2.f : 0x1p-14f;
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          // (2^-14 last: where it makes the product subnormal, the scores are below 2^-90)
          const float f0 = s.ks * qscale[nt][0] * q_unit, f1 = s.ks * qscale[nt][1] * q_unit;
#pragma unroll
          for (int i = 0; i < kTC; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[i][nt][e] *= (e & 1) ? f1 : f0;
        }
        if (s.flags & kMasked) {  // (a ring step is)
          const int pos0 = s.pos0 + round * H::kTok, hi = ring ? 8 + g : 8 + (g ^ 4);
          const int n0 = (s.sub - head_of(s.sub) * p.row_tiles) * kRows;
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int limit = limit_at(s.len, s.cnt, n0 + 8 * nt + 2 * t + (e & 1));
#pragma unroll
              for (int i = 0; i < kTC; ++i)
                if ((ring && i >= kRC) || !sees(p, pos0 + 16 * i + (e < 2 ? g : hi), limit)) sc[i][nt][e] = -INFINITY;
            }
        }
        // ---- online softmax, and P as B fragments.  A round's weights are taken
        // relative to its own maximum x and times 2^15, P = 2^(s - x + 15), which
        // uses fp16 from its top on: with the low part, a weight has an error of
        // 2^-22, or of 2^-40 of the round's largest if that is more.  (Relative to
        // the maximum m so far, a long tail of weights below 2^-25 of one large
        // weight would vanish from the sums, but not from l.)  share = 2^(x - 15 - m)
        // brings the round's sums to m.  The bf16 parts beside bf16 tokens have the
        // range, and those tokens' sums no room for 2^15.
        const float raise = kBf16 && ring ? 0.f : 15.f;
        float alpha[kNT][2], share[kNT][2], row_vs[kNT][2];
        // vs * share of a bf16 block with tiny values would be subnormal: they are multiplied in turn
        const bool tiny = kBf16 && s.vs < 0x1p-60f;
        uint32_t pb[kTC][kNT][2], pl[kTC][kNT][2];
        bool moved = false;
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          float ref[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = -INFINITY;
#pragma unroll
            for (int i = 0; i < kTC; ++i) x = fmaxf(x, fmaxf(sc[i][nt][e], sc[i][nt][2 + e]));
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
            const bool none = x == -INFINITY;
            const float mn = fmaxf(m[nt][e], x), to = mn == -INFINITY ? 0.f : mn;
            // (from 2^20 on x - 15 would be rounded: P as it is; a maximum of 2^15.1 at most is left below 65504)
            ref[e] = none ? 0.f : fabsf(x) < 0x1p20f ? x - raise : x;
            share[nt][e] = none ? 0.f : fast_exp2(ref[e] - to);
            // a row that sees nothing of this block takes nothing of it, not even a scale that is NaN
            row_vs[nt][e] = none ? 0.f : tiny ? s.vs : s.vs * share[nt][e];
            alpha[nt][e] = fast_exp2(m[nt][e] - to);
            moved |= alpha[nt][e] != 1.f;
            m[nt][e] = mn;
          }
          float sum[2] = {0.f, 0.f};
#pragma unroll
          for (int i = 0; i < kTC; ++i) {
            const float p0 = fast_exp2(sc[i][nt][0] - ref[0]), p1 = fast_exp2(sc[i][nt][1] - ref[1]);
            const float p2 = fast_exp2(sc[i][nt][2] - ref[0]), p3 = fast_exp2(sc[i][nt][3] - ref[1]);
            sum[0] += p0 + p2;
            sum[1] += p1 + p3;
            uint32_t hi0, hi1, lo0, lo1;
            // P in two parts: as one fp16 number it would add 2^-11 to an output's rounding, which is 2^-11
            // itself in fp16 and 2^-8 in bf16 (and changes a bf16 output's last place in 1 of 40).
            if (kBf16 && ring) {
              split_pair<true>(p0, p1, hi0, lo0);
              split_pair<true>(p2, p3, hi1, lo1);
            } else {
              split_pair<false>(p0, p1, hi0, lo0);
              split_pair<false>(p2, p3, hi1, lo1);
            }
            pb[i][nt][0] = movmatrix_trans(hi0);  // rows 2t, 2t + 1 of the tokens, query row g
            pb[i][nt][1] = movmatrix_trans(hi1);  // and 2t + 8, 2t + 9
            pl[i][nt][0] = movmatrix_trans(lo0);
            pl[i][nt][1] = movmatrix_trans(lo1);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) l[nt][e] = l[nt][e] * alpha[nt][e] + sum[e] * share[nt][e];
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[nt][c][e] *= alpha[nt][e & 1];
        }
        // ---- O^T += share vs V^T P^T
        if (round == 0 && !aborted && !mbar_wait(smem_u32(&sm.v_full[warp]), k & 1, p.err)) aborted = true;
        if (!ring) {
          const uint32_t va = vb + v_off + round * H::kTok * kD;
#pragma unroll
          for (int c = 0; c < kChunks; c += 2) {
            const uint32_t vc = va ^ (c << 4);
            float blk[2][kNT][4];
#pragma unroll
            for (int i = 0; i < kTC; ++i) {
              uint32_t r[4];
              ldmatrix_b8_trans(vc + 16 * i * kD, r[0], r[1], r[2], r[3]);
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                uint32_t a0, a1, a2, a3;
                to_half<kInt8>(r[2 * j], a0, a2);
                to_half<kInt8>(r[2 * j + 1], a1, a3);
#pragma unroll
                for (int nt = 0; nt < kNT; ++nt) {
                  if (i == 0)
                    mma_first(blk[j][nt], a0, a1, a2, a3, pb[i][nt][0], pb[i][nt][1]);
                  else
                    mma_16816(blk[j][nt], a0, a1, a2, a3, pb[i][nt][0], pb[i][nt][1]);
                  mma_16816(blk[j][nt], a0, a1, a2, a3, pl[i][nt][0], pl[i][nt][1]);
                }
              }
            }
            if (tiny) {
#pragma unroll
              for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    blk[j][nt][e] *= share[nt][e & 1];
                    asm volatile("" : "+f"(blk[j][nt][e]));  // (a branch: predicated, all rounds would issue these)
                  }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][c + j][e] += row_vs[nt][e & 1] * blk[j][nt][e];
          }
        } else {
          // (a sum of its own for each 16 tokens: it has to be weighted, and one for both would take more registers)
#pragma unroll
          for (int i = 0; i < kRC; ++i) {
            const int tok0 = round * H::kTok + 16 * i;
            if (tok0 >= n_tok) break;
            // halves of a register are tokens 2t and 2t + 1 (a0, a1) or 2t + 8 and 2t + 9 (a2, a3); where there is
            // no token, whatever the slot held is taken out
            auto keep = [&](int tok) { return (tok < n_tok ? 0xffffu : 0u) | (tok + 1 < n_tok ? 0xffff0000u : 0u); };
            const uint32_t keep0 = keep(tok0 + 2 * t), keep1 = keep(tok0 + 2 * t + 8);
            const uint32_t row = tok0 + (lane >> 4) * 8 + (lane & 7);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
              uint32_t a[4];
              ldmatrix_x4_trans(vb + (c >> 2) * G::kRegion + row * 128 +
                                    ((((c & 3) * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4),
                                a[0], a[1], a[2], a[3]);
              a[0] &= keep0, a[1] &= keep0, a[2] &= keep1, a[3] &= keep1;
              if (s.flags & kUnclean) {
                // Values that are not finite would reach rows that do not see
                // them (0 * NaN).  They are taken out, and a product of their
                // places with the rows' masks says which sums they make NaN.
                const int h = head_of(s.sub), n0 = (s.sub - h * p.row_tiles) * kRows;
                const uint32_t one = kBf16 ? 0x3f803f80u : 0x3c003c00u;
                uint32_t at[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t mk = nonfinite_mask<kBf16>(a[e]);
                  at[e] = one & mk;
                  a[e] &= ~mk;
                }
#pragma unroll
                for (int nt = 0; nt < kNT; ++nt) {
                  const int lim = limit_at(s.len, s.cnt, n0 + 8 * nt + g);
                  uint32_t see[2];
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const int pos = s.pos0 + tok0 + 2 * t + 8 * e;
                    see[e] = one & ((sees(p, pos, lim) ? 0xffffu : 0u) | (sees(p, pos + 1, lim) ? 0xffff0000u : 0u));
                  }
                  float hit[4] = {0.f, 0.f, 0.f, 0.f};
                  mma_elem<kBf16>(hit, at[0], at[1], at[2], at[3], see[0], see[1]);
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    if (hit[e] > 0.f) acc[nt][c][e] = NAN;
                }
              }
#pragma unroll
              for (int nt = 0; nt < kNT; ++nt) {
                float blk[4] = {0.f, 0.f, 0.f, 0.f};
                mma_elem<kBf16>(blk, a[0], a[1], a[2], a[3], pb[i][nt][0], pb[i][nt][1]);
                mma_elem<kBf16>(blk, a[0], a[1], a[2], a[3], pl[i][nt][0], pl[i][nt][1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][c][e] += share[nt][e & 1] * blk[e];
              }
            }
          }
        }
      }
    }
    __syncwarp();
    issue(k + 1, true);

    if (!(s.flags & kLast)) continue;
    // ---- end of the piece
    const int h = head_of(s.sub), n0 = (s.sub - h * p.row_tiles) * kRows;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], off);
    if (begins && (s.flags & kEnd)) {
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        float inv[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tok = token_of(p, min(n0 + 8 * nt + 2 * t + e, p.rows - 1));
          inv[e] = (l[nt][e] == 0.f || tok >= s.cnt) ? 0.f : 1.f / l[nt][e];
        }
        // dims g of rows 2t, 2t + 1 become dims 2t, 2t + 1 of row g
        const int n = n0 + 8 * nt + g, tok = token_of(p, min(n, p.rows - 1));
        uint16_t* out = p.o.row(s.b, h * p.group + n - tok * p.group, tok) + 2 * t;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const uint32_t x = movmatrix_trans(
                Elem<kBf16>::pack(inv[0] == 0.f ? 0.f : acc[nt][c][e] * inv[0],
                                  inv[1] == 0.f ? 0.f : acc[nt][c][e + 1] * inv[1]));
            if (n < p.rows) *reinterpret_cast<uint32_t*>(out + 16 * c + 4 * e) = x;
          }
      }
      continue;
    }
    // a part of a unit: left for the CTA's end (in the worker's stages after its last step, where it fits)
    constexpr bool kFits = kPiece * 4 <= sizeof(sm.stage[0]);
    float* data = kFits && k == n_steps - 1 ? reinterpret_cast<float*>(sm.stage[warp])
                                   : p.partials + (int64_t(worker) * 2 + (begins ? 1 : 0)) * kPiece;
    if (lane == 0)
      sm.part[warp][begins ? 1 : 0] = Part{x0 + k - s.step, data, s.b, s.sub, s.cnt, s.steps,
                                           kFirst | (begins ? kBegin : 0) | (s.flags & kEnd)};
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * nt + 2 * t + e;
        if (g == 0) reinterpret_cast<float2*>(data)[r] = make_float2(m[nt][e], l[nt][e]);
        float* o = data + 2 * kRows + r * kD + g;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          o[16 * c] = acc[nt][c][e];
          o[16 * c + 8] = acc[nt][c][2 + e];
        }
      }
  }

  // ---- cut units.  The CTA's parts in order (entry 2w + slot: slot 0 goes on
  // from the worker before, slot 1 begins a unit) form runs, one per unit.
  __syncthreads();
  const int e_flags = lane < 2 * H::kWarps ? sm.part[lane >> 1][lane & 1].flags : 0;
  const uint32_t valid = __ballot_sync(0xffffffffu, e_flags != 0);
  if (valid == 0) return;
  const uint32_t begin_mask = __ballot_sync(0xffffffffu, e_flags & kBegin), end_mask = __ballot_sync(0xffffffffu, e_flags & kEnd);
  const uint32_t run_starts = begin_mask | (valid & -valid);
  constexpr int kCols = kD / 32;
  auto store_row = [&](const Part& u, int row, float L, const float (&a)[kCols]) {
    const int h = head_of(u.sub), n = (u.sub - h * p.row_tiles) * kRows + row;
    if (n >= p.rows) return;
    const int tok = token_of(p, n);
    const float inv = (L == 0.f || tok >= u.cnt) ? 0.f : 1.f / L;
    uint16_t* out = p.o.row(u.b, h * p.group + n - tok * p.group, tok) + lane * kCols;
#pragma unroll
    for (int k = 0; k < kCols; k += 2)
      *reinterpret_cast<uint32_t*>(out + k) = inv == 0.f ? 0u : Elem<kBf16>::pack(a[k] * inv, a[k + 1] * inv);
  };
  float* const cta_parts = p.partials + int64_t(gridDim.x) * H::kWarps * 2 * kPiece;
  int cut[2] = {-1, -1};  // first entries of the runs that other CTAs share: going on from one, and begun here
  int task = 0;
  for (uint32_t left = run_starts; left; left &= left - 1) {
    const int first = __ffs(left) - 1;
    const uint32_t later = left & (left - 1);
    const uint32_t in_run = valid & ~((1u << first) - 1u) & (later ? (later & -later) - 1u : 0xffffffffu);
    const int last = 31 - __clz(in_run), n = __popc(in_run);
    const bool b = (begin_mask >> first) & 1, whole = b && ((end_mask >> last) & 1);
    if (!whole) cut[b] = first;
    const Part u = sm.part[first >> 1][first & 1];
    for (int row = 0; row < kRows; ++row, ++task) {
      if (task % H::kWarps != warp) continue;
      float M, L, a[kCols];
      // entries of a run: its first, then slot 0 of the workers behind
      merge_row<kD, kRows, false>(n, row, lane, [&](int i) {
        return const_cast<const float*>(i == 0 ? sm.part[first >> 1][first & 1].data : sm.part[(first >> 1) + i][0].data);
      }, M, L, a);
      if (whole) {
        store_row(u, row, L, a);
      } else {
        float* data = cta_parts + (int64_t(blockIdx.x) * 2 + b) * kPiece;
        if (lane == 0) __stcg(reinterpret_cast<float2*>(data) + row, make_float2(M, L));
        float* o = data + 2 * kRows + row * kD + lane * kCols;
#pragma unroll
        for (int k = 0; k < kCols; k += 2) __stcg(reinterpret_cast<float2*>(o + k), make_float2(a[k], a[k + 1]));
      }
    }
  }
  if (cut[0] < 0 && cut[1] < 0) return;
  __syncthreads();
  // (borders inside a cut unit are where the split put them)
  auto cta_of = [&](int x) { return static_cast<int>(split.owner(x)); };
  if (tid < 2) {
    sm.last[tid] = 0;
    const int c = tid ? cut[1] : cut[0];
    if (c >= 0) {
      const Part& u = sm.part[c >> 1][c & 1];
      const int c0 = cta_of(u.unit_begin), c1 = cta_of(u.unit_begin + u.steps - 1);
      // the barrier above and this fence order the CTA's stores before its ticket
      __threadfence();
      sm.last[tid] = atomicAdd(p.tickets + c0, 1) == c1 - c0;
      __threadfence();
      if (sm.last[tid]) p.tickets[c0] = 0;  // ready for the next launch
    }
  }
  __syncthreads();
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    if (!sm.last[side]) continue;
    const Part u = sm.part[cut[side] >> 1][cut[side] & 1];
    const int c0 = cta_of(u.unit_begin), c1 = cta_of(u.unit_begin + u.steps - 1);
    // the first CTA's part begins there, the others' go on from the one before
    for (int row = warp; row < kRows; row += H::kWarps) {
      float M, L, a[kCols];
      merge_row<kD, kRows, true>(c1 - c0 + 1, row, lane, [&](int i) {
        return const_cast<const float*>(cta_parts + (int64_t(c0 + i) * 2 + (i == 0)) * kPiece);
      }, M, L, a);
      store_row(u, row, L, a);
    }
  }
}

struct Plan {
  int nt, row_tiles, n_ctas;
  size_t bytes;
};

int max_ctas() {
  const int sms = current_device().sm_count;
  return sms > 0 ? sms : 148;
}

// Query rows of a unit: 8 or 16; more of them are further units.
Plan plan(const nsa_kv8_cache* c, int64_t rows) {
  Plan s;
  s.nt = rows <= 8 ? 1 : 2;
  const int tile = 8 * s.nt;
  const int workers = s.nt * c->head_dim <= 128 ? Shape<128, 1>::kWarps : Shape<128, 2>::kWarps;
  s.row_tiles = static_cast<int>((rows + tile - 1) / tile);
  const int64_t most = c->batch * c->n_kv_heads * s.row_tiles * (c->max_blocks + 2);  // steps
  s.n_ctas = static_cast<int>(most < max_ctas() ? most : max_ctas());
  s.bytes = size_t(s.n_ctas) * (workers + 1) * 2 * tile * (2 + c->head_dim) * sizeof(float);
  return s;
}

template <int kD, int kNT, bool kBf16, bool kInt8>
int launch_attend(const Plan& plan, const CUtensorMap (&maps)[4], const AttendParams& p, cudaStream_t stream) {
  using S = Smem<kD, kNT>;
  using H = Shape<kD, kNT>;
  static_assert(offsetof(S, stage) == 0 && Geo<kD>::kHalf % 1024 == 0, "TMA destinations");
  static_assert(offsetof(S, q) % 16 == 0, "vector reads");
  static_assert(sizeof(S) <= 227 * 1024, "shared memory of an SM");
  static_assert(2 * H::kWarps <= 32, "a lane for each part");
  auto kernel = kv8_attend_kernel<kD, kNT, kBf16, kInt8>;
  static bool attr_set[64] = {false};
  const int dev = current_device().device;
  if (dev < 0 || dev >= 64) return fail(NSA_ERR_CUDA, "no CUDA device");
  if (!attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(S)));
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    attr_set[dev] = true;
  }
  cudaError_t e = launch_kernel(kernel, dim3(plan.n_ctas), dim3(H::kThreads), sizeof(S), stream, maps[0], maps[1],
                                maps[2], maps[3], p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? NSA_OK : cuda_fail(e, "kv8_attend_kernel launch");
}

template <int kD, bool kBf16, bool kInt8>
int launch_rows(const Plan& s, const CUtensorMap (&maps)[4], const AttendParams& p, cudaStream_t stream) {
  if (s.nt == 1) return launch_attend<kD, 1, kBf16, kInt8>(s, maps, p, stream);
  return launch_attend<kD, 2, kBf16, kInt8>(s, maps, p, stream);
}

int check_shape(const nsa_kv8_cache* cache, int64_t n_heads, int64_t n_tokens) {
  if (n_heads < 1 || n_heads % cache->n_kv_heads)
    return fail(NSA_ERR_INVALID, "n_heads must be a positive multiple of n_kv_heads (%lld)", (long long)cache->n_kv_heads);
  if (n_heads / cache->n_kv_heads > 1024) return fail(NSA_ERR_UNSUPPORTED, "at most 1024 query heads per KV head");
  if (n_tokens < 1 || n_tokens > kMaxQuery)
    return fail(NSA_ERR_INVALID, "n_tokens must be in [1, %d], got %lld", kMaxQuery, (long long)n_tokens);
  return NSA_OK;
}

}  // namespace
}  // namespace kv8
}  // namespace nsa

using namespace nsa;

extern "C" {

int64_t nsa_kv8_ticket_count(void) { return kv8::max_ctas(); }

size_t nsa_kv8_workspace_bytes(const nsa_kv8_cache* cache, int64_t n_heads, int64_t n_tokens) {
  clear_error();
  kv8::Cache c;
  if (kv8::check_cache(cache, c) || kv8::check_shape(cache, n_heads, n_tokens)) return 0;
  return kv8::plan(cache, n_heads / cache->n_kv_heads * n_tokens).bytes;
}

}  // extern "C"

namespace {

// The append that comes with an attention in a decode step.
struct Append {
  const nsa_kv8_rows *new_k, *new_v;
  const int64_t* starts;
};

// Checks an attention's arguments, then runs the append (if any; nothing is
// written when an argument of either is refused) and launches the attention.
int attend(const nsa_kv8_cache* cache, const Append* add, const nsa_kv8_rows* q, const nsa_kv8_rows* o, int64_t n_heads,
           int64_t n_tokens, const int64_t* counts, int64_t window, int64_t sink, float sm_scale, void* workspace,
           size_t workspace_bytes, int32_t* tickets, nsa_stream_t stream) {
  kv8::AttendParams p{};
  int rc = kv8::check_cache(cache, p.c);
  if (rc) return rc;
  if ((rc = kv8::check_shape(cache, n_heads, n_tokens))) return rc;
  if (sink < 0 || sink > kv8::kMaxPos || window > kv8::kMaxPos)
    return fail(NSA_ERR_INVALID, "need 0 <= sink <= 2^30 and window <= 2^30");
  if (!(sm_scale - sm_scale == 0.f)) return fail(NSA_ERR_INVALID, "sm_scale must be finite");
  if (p.c.batch == 0) return NSA_OK;
  if ((rc = kv8::check_rows(q, "q", p.q))) return rc;
  if ((rc = kv8::check_rows(o, "o", p.o))) return rc;
  p.group = static_cast<int>(n_heads / cache->n_kv_heads);
  p.n_tokens = static_cast<int>(n_tokens);
  p.rows = p.group * p.n_tokens;
  const kv8::Plan s = kv8::plan(cache, p.rows);
  if (int64_t(p.c.n_kv_heads) * s.row_tiles * (int64_t(p.c.max_blocks) + 2) > 0x7fffffff)
    return fail(NSA_ERR_UNSUPPORTED, "too many (head, block) pairs in a sequence");
  if (!workspace || workspace_bytes < s.bytes)
    return fail(NSA_ERR_WORKSPACE, "workspace of %zu bytes required (got %zu)", s.bytes, workspace ? workspace_bytes : size_t(0));
  if (!aligned16(workspace)) return fail(NSA_ERR_ALIGN, "workspace must be 16-byte aligned");
  if (!tickets) return fail(NSA_ERR_WORKSPACE, "tickets must not be NULL");
  p.row_tiles = s.row_tiles;
  p.units_inv = 1.f / (float(p.c.n_kv_heads) * s.row_tiles);
  p.counts = counts;
  p.window = window < 0 ? -1 : static_cast<int>(window);
  p.sink = static_cast<int>(sink);
  p.scale_log2 = sm_scale * kv8::kLog2e;
  p.group_inv = p.group > 1 ? static_cast<uint32_t>(((uint64_t(1) << 32) + p.group - 1) / p.group) : 0;
  p.tickets = tickets;
  p.partials = static_cast<float*>(workspace);
  p.err = device_error_word();
  if (!p.err) return fail(NSA_ERR_CUDA, "device error word unavailable");

  const uint64_t d = static_cast<uint64_t>(cache->head_dim);
  const uint64_t code_dims[2] = {d, static_cast<uint64_t>(p.c.n_pages) * p.c.n_kv_heads * kv8::kBlock};
  const uint64_t ring_dims[2] = {d, static_cast<uint64_t>(p.c.batch) * p.c.n_kv_heads * kv8::kRing};
  const uint64_t code_stride[1] = {d}, ring_stride[1] = {2 * d};
  const uint32_t code_box[2] = {static_cast<uint32_t>(d), kv8::kBlock}, ring_box[2] = {64, 8};
  const CUtensorMapSwizzle swz = d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  CUtensorMap maps[4];
  const void* base[4] = {p.c.k_codes, p.c.v_codes, p.c.k_ring, p.c.v_ring};
  for (int i = 0; i < 4; ++i) {
    rc = i < 2 ? encode_tiled(&maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base[i], code_dims, code_stride, code_box, swz)
               : encode_tiled(&maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, base[i], ring_dims, ring_stride, ring_box,
                              CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  if (add && (rc = nsa_kv8_append(cache, add->new_k, add->new_v, n_tokens, add->starts, counts, stream))) return rc;
  const bool bf16 = cache->dtype == 2, int8 = cache->codes == NSA_KV8_INT8;
  if (d == 128)
    return bf16 ? (int8 ? kv8::launch_rows<128, true, true>(s, maps, p, stream)
                        : kv8::launch_rows<128, true, false>(s, maps, p, stream))
                : (int8 ? kv8::launch_rows<128, false, true>(s, maps, p, stream)
                        : kv8::launch_rows<128, false, false>(s, maps, p, stream));
  return bf16 ? (int8 ? kv8::launch_rows<64, true, true>(s, maps, p, stream)
                      : kv8::launch_rows<64, true, false>(s, maps, p, stream))
              : (int8 ? kv8::launch_rows<64, false, true>(s, maps, p, stream)
                      : kv8::launch_rows<64, false, false>(s, maps, p, stream));
}

}  // namespace

extern "C" {

int nsa_kv8_attend(const nsa_kv8_cache* cache, const nsa_kv8_rows* q, const nsa_kv8_rows* o, int64_t n_heads,
                   int64_t n_tokens, const int64_t* counts, int64_t window, int64_t sink, float sm_scale,
                   void* workspace, size_t workspace_bytes, int32_t* tickets, nsa_stream_t stream) {
  clear_error();
  return attend(cache, nullptr, q, o, n_heads, n_tokens, counts, window, sink, sm_scale, workspace, workspace_bytes,
                tickets, stream);
}

int nsa_kv8_decode_step(const nsa_kv8_cache* cache, const nsa_kv8_rows* new_k, const nsa_kv8_rows* new_v,
                        const nsa_kv8_rows* q, const nsa_kv8_rows* o, int64_t n_heads, int64_t n_tokens,
                        const int64_t* starts, const int64_t* counts, int64_t window, int64_t sink, float sm_scale,
                        void* workspace, size_t workspace_bytes, int32_t* tickets, nsa_stream_t stream) {
  clear_error();
  const Append add{new_k, new_v, starts};
  return attend(cache, &add, q, o, n_heads, n_tokens, counts, window, sink, sm_scale, workspace, workspace_bytes,
                tickets, stream);
}

}  // extern "C"
