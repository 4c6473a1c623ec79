// Attention over the 8-bit paged cache, for the last 1 to 64 tokens of every
// sequence (decode, verification of drafts).
//
//   o[n] = sum_p softmax_p(scale * q[n] . k[p]) v[p],  k[p] = ks(block of p) * kc[p], v likewise
//
// The scales leave the products: s = ks * (q . kc), o = sum over blocks of
// vs * (P . vc).  The codes become fp16 exactly (e4m3 and int8 both fit), so the
// products run on mma.sync m16n8k16 with fp16 operands and fp32 sums.  Queries
// enter as fp16 after a power of two per row has brought their largest element
// into [1, 2): exact for fp16 and for bf16 but for elements 2^-14 below the
// row's largest, which keep an absolute error of 2^-25 of it.
//
// Bound by HBM for up to about 32 query rows a KV head: 8 rows take 16 FLOP a
// byte.  tcgen05 would want the codes as fp16 in shared memory first and tiles
// of 64 or 128 rows; here the conversion happens in registers on the way from
// ldmatrix to the mma.
//
// Work is split evenly over persistent CTAs (two per SM) by items: an item is
// a block of 64 tokens, or a sequence's incomplete block (from the ring).  The
// lengths live on the device, so every CTA computes the split itself (one scan
// over the batch).  A CTA's consecutive items form pieces of units (sequence,
// KV head, 32-row tile); a unit cut between CTAs is merged by the last of them to
// finish.  In a CTA one warp feeds a ring of TMA stages and four consume:
// a warp scores 16 of an item's 64 tokens for all rows, the four agree on the rows'
// maxima and exchange P through shared memory, and each accumulates a quarter
// of the head dimension over all 64 tokens.  So the accumulators of a piece
// need no merge between warps (short sequences end often), and they stay at
// 8 registers per 8 rows.
#include <cstddef>
#include <cstdlib>

#include "kv8.cuh"

namespace nsa {
namespace kv8 {
namespace {

constexpr int kWarps = 4;  // consumers
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kCtasPerSm = 2;
constexpr int kRowTile = 32;   // query rows of a unit at most
constexpr int kLensCached = 512;  // sequence lengths kept in shared memory
constexpr float kLog2e = 1.4426950408889634f;

struct AttendParams {
  Cache c;
  Rows q, o;
  int group, n_tokens, rows, row_tiles;  // rows = n_tokens * group of a KV head
  const int64_t* counts;
  int window, sink;  // window < 0: all positions
  float scale_log2;
  int n_ctas;
  int* tickets;    // [n_ctas]
  float* partials;  // [n_ctas][2] pieces of 8 * NT rows: m, l, then kD sums a row
  int* err;
};

// One sequence as the kernel sees it.
struct Seq {
  int len, cnt;       // tokens; query tokens (rows of later ones are 0)
  int full;           // complete blocks
  int sink_blocks, win_block;  // block items: [0, sink_blocks), [win_block, full)
  int items;          // at least 1
  bool empty;         // nothing to see: its one item writes zeros
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
  s.items = s.sink_blocks + s.full - s.win_block + (len % kBlock != 0);
  s.empty = cnt == 0 || s.items == 0;
  if (s.empty) s.items = 1;
  return s;
}

// A sequence's length and query count as one word (both checked): an invalid
// length reads as an empty sequence.
__device__ __forceinline__ int2 load_len(const AttendParams& p, int b) {
  const int64_t len = p.c.lens[b];
  const int64_t cnt = p.counts ? p.counts[b] : p.n_tokens;
  if (len < 0 || len > int64_t(p.c.max_blocks) * kBlock || cnt < 0 || cnt > p.n_tokens) {
    set_error(p.err, NSA_ERR_INVALID);
    return make_int2(0, 0);
  }
  return make_int2(static_cast<int>(len), static_cast<int>(cnt));
}

template <int kD>
struct Geo {
  static constexpr uint32_t kCodeBytes = kBlock * kD;         // K (or V) codes of a block
  static constexpr uint32_t kStageBytes = 2 * kCodeBytes;     // also 32 ring tokens of K and V
  static constexpr uint32_t kRegions = kD / 64;               // 128-byte column halves of a ring tile
  static constexpr uint32_t kRegion = 32 * 128;               // 32 ring rows of one half
  static constexpr int kQStride = kD * 2 + 32;                // bytes: rows 8 banks apart
};

constexpr int kPStride = kBlock * 2 + 16;  // bytes of a row of P: rows 4 banks apart

template <int kD, int kNT>
struct Smem {
  static constexpr int kStages = (kNT == 1 ? 6 : 5) * (128 / kD);  // 80-96 KiB in flight a CTA
  uint8_t stage[kStages][Geo<kD>::kStageBytes];  // 1024-aligned: TMA destinations
  uint8_t q[2][8 * kNT][Geo<kD>::kQStride];
  uint8_t p_hi[8 * kNT][kPStride];
  uint8_t p_lo[8 * kNT][kPStride];
  float q_scale[8 * kNT];
  float mx[kWarps][8 * kNT];  // rows' maxima over each warp's tokens; sums at a piece's end
  float2 scale[kStages];
  int2 lens[kLensCached];
  int scan[kThreads / 32];
  int b0, base_hi, base_lo;  // first sequence of this CTA, items before it
  int ticket;
  uint64_t full[kStages], empty[kStages];
  uint64_t q_full[2], q_empty[2];
};

__device__ __forceinline__ void sync_consumers() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); }

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

// Four codes to two fp16 pairs: (bytes 0, 1) and (2, 3), or with kSplit
// (0, 2) and (1, 3).  int8: the byte, biased by 128, is the low part of an
// fp16 number in [1024, 2048), from which 1152 is taken again (exact).
template <bool kInt8, bool kSplit>
__device__ __forceinline__ void to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kInt8) {
    const uint32_t x = w ^ 0x80808080u, magic = 0x64646464u;
    const uint32_t a = __byte_perm(x, magic, kSplit ? 0x4240 : 0x4140);
    const uint32_t b = __byte_perm(x, magic, kSplit ? 0x4341 : 0x4342);
    const __half2 bias = __float2half2_rn(1152.f);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&a), bias);
    const __half2 z = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
    lo = *reinterpret_cast<const uint32_t*>(&y);
    hi = *reinterpret_cast<const uint32_t*>(&z);
  } else {
    const uint32_t x = kSplit ? __byte_perm(w, 0u, 0x3120) : w;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(x));
  }
}

__device__ __forceinline__ void lds8(uint32_t addr, uint32_t& lo, uint32_t& hi) {
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(lo), "=r"(hi) : "r"(addr));
}
__device__ __forceinline__ uint32_t lds4(uint32_t addr) {
  uint32_t x;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(addr));
  return x;
}

// Stores x as a 16-bit number at byte `at` of p_hi and, with `split`, what
// that rounding left at `at` of p_lo.
template <bool kBf16, class SmemT>
__device__ __forceinline__ void store_p(SmemT& sm, uint32_t at, float x, bool split) {
  uint8_t* hi = &sm.p_hi[0][0] + at;
  uint8_t* lo = &sm.p_lo[0][0] + at;
  if constexpr (kBf16) {
    const __nv_bfloat16 y = __float2bfloat16_rn(x);
    *reinterpret_cast<__nv_bfloat16*>(hi) = y;
    if (split) *reinterpret_cast<__nv_bfloat16*>(lo) = __float2bfloat16_rn(x - __bfloat162float(y));
  } else {
    const __half y = __float2half_rn(x);
    *reinterpret_cast<__half*>(hi) = y;
    if (split) *reinterpret_cast<__half*>(lo) = __float2half_rn(x - __half2float(y));
  }
}

// A pair of fp16 numbers of 8 significant bits as bf16 (exact).  volatile, so
// that the conversions of all query fragments stay on the ring's path instead
// of being kept in registers.
__device__ __forceinline__ uint32_t half_to_bf16(uint32_t x) {
  uint32_t y;
  asm volatile(
      "{\n\t.reg .b16 l, h;\n\t.reg .f32 a, b;\n\tmov.b32 {l, h}, %1;\n\tcvt.f32.f16 a, l;\n\tcvt.f32.f16 b, h;\n\t"
      "cvt.rn.bf16x2.f32 %0, b, a;\n\t}"
      : "=r"(y)
      : "r"(x));
  return y;
}

// Whether a row with position limit `lim` sees `pos`.
__device__ __forceinline__ bool sees(const AttendParams& p, int pos, int lim) {
  return pos < lim && (p.window < 0 || pos < p.sink || pos >= lim - p.window);
}

// The values of an incomplete block (ring slots in stages st and st1, 32
// each; `tail` of them hold tokens, pos0 is the first's position) times P, for
// the warp's head dimensions: blk = V^T P^T.  Rows of P are split in two.
template <int kD, int kNT, bool kBf16, class SmemT, class LimitOf>
__device__ __forceinline__ void ring_values(const SmemT& sm, const AttendParams& p, uint32_t st, uint32_t st1, int tail,
                                            int pos0, int warp, int lane, LimitOf limit_of, int n0, uint32_t ph,
                                            uint32_t pl, float (&blk)[kNT][kD / 64][4]) {
  using G = Geo<kD>;
  constexpr int kMT = kD / 64;
  const int g = lane >> 2, t = lane & 3;
  for (int kk = 0; kk < 2 && 32 * kk < tail; ++kk) {
    const uint32_t vb = smem_u32(sm.stage[kk ? st1 : st]) + G::kCodeBytes;
    uint32_t a[2][kMT][4];
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < kMT; ++c) {
        const int cc = kMT * warp + c;  // 16-wide chunk of the head dimension
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // tokens 2t, 2t + 1, 2t + 8, 2t + 9: dims 2g, 2g + 1
          const uint32_t row = 16 * i + 2 * t + (e & 1) + (e >> 1) * 8;
          w[e] = lds4(vb + (cc >> 2) * G::kRegion + row * 128 + ((((cc & 3) * 2 + (g >> 2)) ^ (row & 7)) << 4) +
                      (g & 3) * 4);
          if (32 * kk + static_cast<int>(row) >= tail) w[e] = 0u;  // no token: whatever the slot held
          bad |= nonfinite_mask<kBf16>(w[e]);
        }
        a[i][c][0] = __byte_perm(w[0], w[1], 0x5410);
        a[i][c][1] = __byte_perm(w[0], w[1], 0x7632);
        a[i][c][2] = __byte_perm(w[2], w[3], 0x5410);
        a[i][c][3] = __byte_perm(w[2], w[3], 0x7632);
      }
    const bool any_bad = __any_sync(0xffffffffu, bad != 0);
    if (any_bad) {
      // Values that are not finite would reach rows that do not see them (0 *
      // NaN).  They are taken out, and a product of their places with the
      // rows' masks says which sums they make NaN.
      const uint32_t one = kBf16 ? 0x3f803f80u : 0x3c003c00u;
      uint32_t ind[2][kMT][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < kMT; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t mk = nonfinite_mask<kBf16>(a[i][c][e]);
            ind[i][c][e] = one & mk;
            a[i][c][e] &= ~mk;
          }
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        const int lim = limit_of(n0 + 8 * nt + g);
        float hit[kMT][4];
#pragma unroll
        for (int c = 0; c < kMT; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) hit[c][e] = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t b[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int pos = pos0 + 32 * kk + 16 * i + 2 * t + 8 * e;
            b[e] = one & ((sees(p, pos, lim) ? 0xffffu : 0u) | (sees(p, pos + 1, lim) ? 0xffff0000u : 0u));
          }
#pragma unroll
          for (int c = 0; c < kMT; ++c)
            mma_elem<kBf16>(hit[c], ind[i][c][0], ind[i][c][1], ind[i][c][2], ind[i][c][3], b[0], b[1]);
        }
#pragma unroll
        for (int c = 0; c < kMT; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (hit[c][e] > 0.f) blk[nt][c][e] = NAN;
      }
    }
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      uint32_t b[4], b2[4];
      ldmatrix_x4(ph + nt * 8 * kPStride + kk * 64, b[0], b[1], b[2], b[3]);
      ldmatrix_x4(pl + nt * 8 * kPStride + kk * 64, b2[0], b2[1], b2[2], b2[3]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < kMT; ++c) {
          mma_elem<kBf16>(blk[nt][c], a[i][c][0], a[i][c][1], a[i][c][2], a[i][c][3], b[2 * i], b[2 * i + 1]);
          mma_elem<kBf16>(blk[nt][c], a[i][c][0], a[i][c][1], a[i][c][2], a[i][c][3], b2[2 * i], b2[2 * i + 1]);
        }
    }
  }
}

// The even split of `total` items over n CTAs: CTA c takes [c, c + 1) * total / n.
__device__ __forceinline__ int64_t split_at(int64_t c, int64_t total, int64_t n) { return c * total / n; }
__device__ __forceinline__ int owner(int64_t x, int64_t total, int64_t n) {
  return static_cast<int>(((x + 1) * n + total - 1) / total - 1);
}

// Walks the pieces of a CTA's items [x, x_end): a run of one unit's items.
struct Pieces {
  int64_t x, x_end, unit_begin;
  int b, sub;  // sequence; KV head * row_tiles + row tile
  Seq s;
  int begin, end;  // items of the unit

  template <class SmemT>
  __device__ __forceinline__ void load(const AttendParams& p, const SmemT& sm) {
    const int2 l = b < kLensCached ? sm.lens[b] : load_len(p, b);
    s = make_seq(p, l.x, l.y);
  }
  template <class SmemT>
  __device__ __forceinline__ void init(const AttendParams& p, const SmemT& sm, int64_t x0, int64_t x1) {
    x = x0;
    x_end = x1;
    b = sm.b0;
    const int64_t base = (int64_t(sm.base_hi) << 32) | static_cast<uint32_t>(sm.base_lo);
    load(p, sm);
    sub = static_cast<int>((x - base) / s.items);
    unit_begin = base + int64_t(sub) * s.items;
    begin = end = 0;
  }
  // The next piece, or false.
  template <class SmemT>
  __device__ __forceinline__ bool next(const AttendParams& p, const SmemT& sm) {
    if (x >= x_end) return false;
    if (x == unit_begin + s.items) {
      unit_begin = x;
      if (++sub == p.c.n_kv_heads * p.row_tiles) {
        sub = 0;
        ++b;
        load(p, sm);
      }
    }
    begin = static_cast<int>(x - unit_begin);
    end = static_cast<int>(min(x_end - unit_begin, int64_t(s.items)));
    x = unit_begin + end;
    return true;
  }
  __device__ __forceinline__ int blocks() const { return s.sink_blocks + s.full - s.win_block; }
  __device__ __forceinline__ int block_of(int item) const {
    return item < s.sink_blocks ? item : s.win_block + item - s.sink_blocks;
  }
};

template <int kD, int kNT, bool kBf16, bool kInt8>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    kv8_attend_kernel(const __grid_constant__ CUtensorMap tm_kc, const __grid_constant__ CUtensorMap tm_vc,
                      const __grid_constant__ CUtensorMap tm_kr, const __grid_constant__ CUtensorMap tm_vr,
                      const AttendParams p) {
  using G = Geo<kD>;
  using S = Smem<kD, kNT>;
  constexpr int kStages = S::kStages;
  constexpr int kChunks = kD / 16;      // 16-wide steps of the head dimension
  constexpr int kMT = kChunks / kWarps;  // those that a warp accumulates
  constexpr int kRows = 8 * kNT;
  // P as one fp16 number has a relative error of 2^-12, the same as rounding
  // the output to fp16 makes, and far below bf16's.  With fp16 outputs P is
  // the sum of two fp16 numbers (2^-23); the memory-bound loop has room for it.
  constexpr bool kSplitP = !kBf16;
  // Query fragments of 32 rows of 128 would take 64 registers a thread (of 168 that
  // two CTAs of five warps leave); they are read from shared memory instead.
  constexpr bool kQShared = kNT * kD >= 256;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  grid_launch_dependents();
  if (smem_u32(smem_raw) & 1023u) {
    if (threadIdx.x == 0) set_error(p.err, NSA_ERR_ALIGN);
    return;
  }
  S& sm = *reinterpret_cast<S*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&sm.full[s]), 1);
      mbar_init(smem_u32(&sm.empty[s]), kWarps);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&sm.q_full[s]), 1);
      mbar_init(smem_u32(&sm.q_empty[s]), kWarps);
    }
    fence_barrier_init();
  }
  if (tid == kWarps * 32) {
    prefetch_tmap(&tm_kc);
    prefetch_tmap(&tm_vc);
    prefetch_tmap(&tm_kr);
    prefetch_tmap(&tm_vr);
  }
  grid_dependency_wait();

  // ---- the split: items before each thread's run of sequences
  const int batch = p.c.batch, per = (batch + kThreads - 1) / kThreads;
  const int units = p.c.n_kv_heads * p.row_tiles;  // of a sequence
  int64_t x0, x1, total;
  {
    int mine = 0;  // items of this thread's sequences, per unit of them
    for (int b = tid * per; b < min(batch, (tid + 1) * per); ++b) {
      const int2 l = load_len(p, b);
      if (b < kLensCached) sm.lens[b] = l;
      mine += make_seq(p, l.x, l.y).items;
    }
    int before = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, before, off);
      if (lane >= off) before += y;
    }
    if (lane == 31) sm.scan[warp] = before;
    __syncthreads();
    int sum = 0, prior = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w == warp) prior = sum;
      sum += sm.scan[w];
    }
    before += prior - mine;
    total = int64_t(sum) * units;
    const int64_t n = min(int64_t(p.n_ctas), total);
    x0 = split_at(blockIdx.x, total, n);
    x1 = split_at(blockIdx.x + 1, total, n);
    if (blockIdx.x >= n) return;  // the same for the whole CTA
    const int64_t lo = int64_t(before) * units, hi = int64_t(before + mine) * units;
    if (x0 >= lo && x0 < hi) {
      int64_t at = lo;
      for (int b = tid * per;; ++b) {
        const int2 l = b < kLensCached ? sm.lens[b] : load_len(p, b);
        const int64_t w = int64_t(make_seq(p, l.x, l.y).items) * units;
        if (x0 < at + w) {
          sm.b0 = b;
          sm.base_hi = static_cast<int>(at >> 32);
          sm.base_lo = static_cast<int>(at);
          break;
        }
        at += w;
      }
    }
    __syncthreads();
  }
  const int64_t n_split = min(int64_t(p.n_ctas), total);

  Pieces pc;
  pc.init(p, sm, x0, x1);
  int qs = 0;
  uint32_t qphase = 0;
  uint32_t st = 0, phase = 0;  // stage ring position
  auto advance = [&]() {
    if (++st == kStages) st = 0, phase ^= 1;
  };

  if (warp == kWarps) {
    // ------------------------------------------------------------- producer
    bool ok = true;
    while (ok && pc.next(p, sm)) {
      if (pc.s.empty) continue;
      const int h = pc.sub / p.row_tiles, n0 = (pc.sub % p.row_tiles) * kRowTile;
      // queries: one row a lane
      if (lane == 0) ok = mbar_wait(smem_u32(&sm.q_empty[qs]), qphase ^ 1, p.err);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      const int n_rows = min(kRows, p.rows - n0);
      const uint32_t qb = smem_u32(&sm.q_full[qs]);
      if (lane == 0) mbar_arrive_expect_tx(qb, n_rows * kD * 2);
      __syncwarp();
      if (lane < n_rows) {
        const int n = n0 + lane, t = n / p.group;
        bulk_load(smem_u32(sm.q[qs][lane]), p.q.row(pc.b, h * p.group + n - t * p.group, t), kD * 2, qb);
      }
      if (++qs == 2) qs = 0, qphase ^= 1;

      const int blocks = pc.blocks();
      for (int i0 = pc.begin; ok && i0 < min(pc.end, blocks); i0 += 32) {
        int page = 0;
        float2 sc = make_float2(NAN, NAN);
        if (i0 + lane < min(pc.end, blocks)) {  // 32 items' page numbers and scales at once
          page = __ldg(p.c.page_table + int64_t(pc.b) * p.c.max_blocks + pc.block_of(i0 + lane));
          if (page >= 0 && page < p.c.n_pages) {
            sc = __ldg(p.c.scales + int64_t(page) * p.c.n_kv_heads + h);
          } else {
            set_error(p.err, NSA_ERR_INVALID);
            page = 0;
          }
        }
        const int cnt = min(32, min(pc.end, blocks) - i0);
        for (int j = 0; j < cnt; ++j) {
          const int pg = __shfl_sync(0xffffffffu, page, j);
          const float2 s2 = make_float2(__shfl_sync(0xffffffffu, sc.x, j), __shfl_sync(0xffffffffu, sc.y, j));
          if (lane == 0) {
            ok = mbar_wait(smem_u32(&sm.empty[st]), phase ^ 1, p.err);
            if (ok) {
              const uint32_t fb = smem_u32(&sm.full[st]), dst = smem_u32(sm.stage[st]);
              sm.scale[st] = s2;  // published by the arrive
              mbar_arrive_expect_tx(fb, G::kStageBytes);
              const int row = (pg * p.c.n_kv_heads + h) * kBlock;
              tma_load_2d(dst, &tm_kc, fb, 0, row);
              tma_load_2d(dst + G::kCodeBytes, &tm_vc, fb, 0, row);
            }
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) break;
          advance();
        }
      }
      if (ok && pc.end > blocks && pc.s.len % kBlock) {  // the incomplete block: 32 ring slots a stage
        const int tail = pc.s.len % kBlock, slot0 = (pc.s.full * kBlock) % kRing;
        const int unit = pc.b * p.c.n_kv_heads + h;
        for (int f = 0; f < tail; f += 32) {
          if (lane == 0) {
            ok = mbar_wait(smem_u32(&sm.empty[st]), phase ^ 1, p.err);
            if (ok) {
              const uint32_t fb = smem_u32(&sm.full[st]), dst = smem_u32(sm.stage[st]);
              const int boxes = min(4, (tail - f + 7) / 8);  // 8 rows each, only those that hold tokens
              mbar_arrive_expect_tx(fb, boxes * 8 * kD * 4);
              for (int r = 0; r < boxes; ++r)
                for (uint32_t c = 0; c < G::kRegions; ++c) {
                  const uint32_t d = dst + c * G::kRegion + r * 1024;
                  tma_load_2d(d, &tm_kr, fb, c * 64, unit * kRing + slot0 + f + 8 * r);
                  tma_load_2d(d + G::kCodeBytes, &tm_vr, fb, c * 64, unit * kRing + slot0 + f + 8 * r);
                }
            }
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) break;
          advance();
        }
      }
    }
    return;
  }

  // -------------------------------------------------------------- consumers
  // After a wait that ran out (the error word is set) a warp waits no more but
  // keeps its schedule of named barriers, so that no other warp waits for it.
  const int g = lane >> 2, t = lane & 3;
  bool aborted = false;
  uint32_t qf[kQShared ? 1 : kNT][kChunks][2];
  float qscale[kNT][2];  // of rows 8nt + 2t, 8nt + 2t + 1: the row's power of two, sm_scale and log2(e)
  float m[kNT][2], l[kNT][2];
  float acc[kNT][kMT][4];  // dims 16c + 2g (0, 1) and 16c + 2g + 1 (2, 3), rows 2t (0, 2) and 2t + 1 (1, 3)

  while (pc.next(p, sm)) {
    const int h = pc.sub / p.row_tiles, n0 = (pc.sub % p.row_tiles) * kRowTile;
    const Seq s = pc.s;
    const bool nothing = pc.s.empty;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) m[nt][e] = -INFINITY, l[nt][e] = 0.f;
#pragma unroll
      for (int c = 0; c < kMT; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][c][e] = 0.f;
    }
    int limit[kNT][2];  // positions below it are seen
    const int first_pos = s.len - s.cnt + 1;
    auto limit_of = [&](int n) { return max(first_pos + min(min(n, p.rows - 1) / p.group, s.cnt - 1), 0); };
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) limit[nt][e] = limit_of(n0 + 8 * nt + 2 * t + e);
    const int limit_min = limit_of(n0), limit_max = limit_of(n0 + kRows - 1);

    if (!nothing) {
      // ---- queries: fp16 fragments, k index permuted as the codes' ldmatrix gives it
      if (!aborted && !mbar_wait(smem_u32(&sm.q_full[qs]), qphase, p.err)) aborted = true;
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        if (kQShared && nt != warp) continue;  // each warp converts 8 rows for all
        uint2 raw[kChunks];
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          raw[c] = *reinterpret_cast<const uint2*>(&sm.q[qs][8 * nt + g][32 * c + 8 * t]);
          const float2 a = Elem<kBf16>::unpack(raw[c].x), b = Elem<kBf16>::unpack(raw[c].y);
          top = fmaxf(top, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // a power of two from the exponent field; rows of zeros or infinities as they are
        int ex = static_cast<int>(__float_as_uint(top) >> 23);
        ex = (top == 0.f || ex == 255) ? 127 : min(max(ex, 1), 253);
        const float f = __uint_as_float(static_cast<uint32_t>(254 - ex) << 23);
        const float back = __uint_as_float(static_cast<uint32_t>(ex) << 23) * p.scale_log2;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const float2 a = Elem<kBf16>::unpack(raw[c].x), b = Elem<kBf16>::unpack(raw[c].y);
          const uint32_t lo = pack_half2(a.x * f, a.y * f), hi = pack_half2(b.x * f, b.y * f);
          if constexpr (kQShared)
            *reinterpret_cast<uint2*>(&sm.q[qs][8 * nt + g][32 * c + 8 * t]) = make_uint2(lo, hi);
          else
            qf[nt][c][0] = lo, qf[nt][c][1] = hi;
        }
        if constexpr (kQShared) {
          if (t == 0) sm.q_scale[8 * nt + g] = back;
        } else {
          qscale[nt][0] = __shfl_sync(0xffffffffu, back, 8 * t);      // from a lane of row 2t
          qscale[nt][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);  // and of 2t + 1
        }
      }
      if constexpr (kQShared) {
        sync_consumers();
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          const float2 x = *reinterpret_cast<const float2*>(&sm.q_scale[8 * nt + 2 * t]);
          qscale[nt][0] = x.x, qscale[nt][1] = x.y;
        }
      } else {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.q_empty[qs]));
        if (++qs == 2) qs = 0, qphase ^= 1;
      }
    }
    const uint32_t q_at = smem_u32(&sm.q[qs][g][8 * t]);  // kQShared: this lane's fragments
    auto q_frag = [&](int nt, int c, uint32_t& b0, uint32_t& b1) {
      if constexpr (kQShared)
        lds8(q_at + nt * 8 * G::kQStride + 32 * c, b0, b1);
      else
        b0 = qf[nt][c][0], b1 = qf[nt][c][1];
    };

    const int blocks = pc.blocks();
    for (int item = pc.begin; !nothing && item < pc.end; ++item) {
      const bool ring = item >= blocks;  // the incomplete block
      const int pos0 = (ring ? s.full : pc.block_of(item)) * kBlock;
      const int tail = s.len - s.full * kBlock;  // its tokens
      const int stages = ring && tail > 32 ? 2 : 1;
      uint32_t st1 = st + 1, phase1 = phase;  // the second stage of an incomplete block
      if (st1 == kStages) st1 = 0, phase1 ^= 1;
      if (!aborted && !mbar_wait(smem_u32(&sm.full[st]), phase, p.err)) aborted = true;
      if (stages == 2 && !aborted && !mbar_wait(smem_u32(&sm.full[st1]), phase1, p.err)) aborted = true;

      // ---- scores of this warp's 16 tokens, S^T: token g (0, 1), g + 8 (2, 3); rows 2t, 2t + 1
      float sc[kNT][4];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[nt][e] = 0.f;
      float vs = 1.f;
      if (!ring) {
        const float2 scale = sm.scale[st];
        vs = scale.y;
        const uint32_t kb = smem_u32(sm.stage[st]);
        const uint32_t row = 16 * warp + ((lane >> 3) & 1) * 8 + (lane & 7), hi = lane >> 4;
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
          uint32_t r[4];
          const uint32_t chunk = kD == 128 ? ((c + hi) ^ (row & 7)) : ((c + hi) ^ ((row >> 1) & 3));
          ldmatrix_x4(kb + row * kD + chunk * 16, r[0], r[1], r[2], r[3]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t a0, a1, a2, a3;
            to_half<kInt8, false>(r[2 * i], a0, a2);
            to_half<kInt8, false>(r[2 * i + 1], a1, a3);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) {
              uint32_t b0, b1;
              q_frag(nt, c + i, b0, b1);
              mma_16816(sc[nt], a0, a1, a2, a3, b0, b1);
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[nt][e] *= scale.x * qscale[nt][e & 1];
      } else if (16 * warp < tail) {
        const uint32_t kb = smem_u32(sm.stage[warp < 2 ? st : st1]);
        const uint32_t row = 16 * (warp & 1) + g;  // row & 7 == g for both of this lane's rows
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const uint32_t at = kb + (c >> 2) * G::kRegion + ((((c & 3) * 2 + (t >> 1)) ^ g) << 4) + (t & 1) * 8;
          uint32_t a0, a1, a2, a3;
          lds8(at + row * 128, a0, a2);
          lds8(at + (row + 8) * 128, a1, a3);
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) {
            uint32_t b0, b1;
            q_frag(nt, c, b0, b1);
            if constexpr (kBf16) b0 = half_to_bf16(b0), b1 = half_to_bf16(b1);
            mma_elem<kBf16>(sc[nt], a0, a1, a2, a3, b0, b1);
          }
        }
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[nt][e] *= qscale[nt][e & 1];
      }
      // ---- masks, where an edge crosses the block
      const bool masked = ring || pos0 + kBlock > limit_min ||
                          (p.window >= 0 && pos0 < limit_max - p.window && pos0 + kBlock > p.sink);
      if (masked) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int pos = pos0 + 16 * warp + g + (e >> 1) * 8, lim = limit[nt][e & 1];
            if (!sees(p, pos, lim)) sc[nt][e] = -INFINITY;
          }
      }
      // ---- rows' maxima over the 64 tokens
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        float a = fmaxf(sc[nt][0], sc[nt][2]), b = fmaxf(sc[nt][1], sc[nt][3]);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, off));
          b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, off));
        }
        if (g == 0) *reinterpret_cast<float2*>(&sm.mx[warp][8 * nt + 2 * t]) = make_float2(a, b);
      }
      sync_consumers();
      float row_vs[kNT][2];
      bool moved = false;
      float alpha[kNT][2];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        float2 top = *reinterpret_cast<const float2*>(&sm.mx[0][8 * nt + 2 * t]);
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
          const float2 o = *reinterpret_cast<const float2*>(&sm.mx[w][8 * nt + 2 * t]);
          top.x = fmaxf(top.x, o.x);
          top.y = fmaxf(top.y, o.y);
        }
        const float tops[2] = {top.x, top.y};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // a row that sees nothing of this block takes nothing of it, not even a scale that is NaN
          row_vs[nt][e] = tops[e] == -INFINITY ? 0.f : vs;
          const float mn = fmaxf(m[nt][e], tops[e]);
          const float ref = mn == -INFINITY ? 0.f : mn;
          alpha[nt][e] = fast_exp2(m[nt][e] - ref);
          moved |= alpha[nt][e] != 1.f;
          m[nt][e] = mn;
          const float p0 = fast_exp2(sc[nt][e] - ref), p1 = fast_exp2(sc[nt][2 + e] - ref);
          l[nt][e] = l[nt][e] * alpha[nt][e] + (p0 + p1);
          // P[row][token], 16-bit, in one or two parts
          const uint32_t at = (8 * nt + 2 * t + e) * kPStride + (16 * warp + g) * 2;
          if (kBf16 && ring) {
            store_p<true>(sm, at, p0, true);
            store_p<true>(sm, at + 16, p1, true);
          } else {
            store_p<false>(sm, at, p0, kSplitP);
            store_p<false>(sm, at + 16, p1, kSplitP);
          }
        }
      }
      sync_consumers();

      // ---- this warp's head dimensions: O^T += V^T P^T over the 64 tokens
      float blk[kNT][kMT][4];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int c = 0; c < kMT; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) blk[nt][c][e] = 0.f;
      const uint32_t pa = ((lane & 7) * kPStride) + (lane >> 3) * 16;  // ldmatrix: 8 rows of P, 32 tokens
      const uint32_t ph = smem_u32(sm.p_hi) + pa, pl = smem_u32(sm.p_lo) + pa;
      if (!ring) {
        const uint32_t vb = smem_u32(sm.stage[st]) + G::kCodeBytes;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {  // 32 tokens
          uint32_t a[2][kMT][4];          // [16 tokens][chunk]
          if constexpr (kMT == 2) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t row = 32 * kk + 16 * i + ((lane >> 3) & 1) * 8 + (lane & 7);
              const uint32_t chunk = (2 * warp + (lane >> 4)) ^ (row & 7);
              uint32_t r[4];
              ldmatrix_x4_trans(vb + row * kD + chunk * 16, r[0], r[1], r[2], r[3]);
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                to_half<kInt8, true>(r[2 * c], a[i][c][0], a[i][c][1]);
                to_half<kInt8, true>(r[2 * c + 1], a[i][c][2], a[i][c][3]);
              }
            }
          } else {
            const uint32_t row = 32 * kk + lane;
            const uint32_t chunk = warp ^ ((row >> 1) & 3);
            uint32_t r[4];
            ldmatrix_x4_trans(vb + row * kD + chunk * 16, r[0], r[1], r[2], r[3]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              to_half<kInt8, true>(r[2 * i], a[i][0][0], a[i][0][1]);
              to_half<kInt8, true>(r[2 * i + 1], a[i][0][2], a[i][0][3]);
            }
          }
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) {
            uint32_t b[4];
            ldmatrix_x4(ph + nt * 8 * kPStride + kk * 64, b[0], b[1], b[2], b[3]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int c = 0; c < kMT; ++c)
                mma_16816(blk[nt][c], a[i][c][0], a[i][c][1], a[i][c][2], a[i][c][3], b[2 * i], b[2 * i + 1]);
            if constexpr (kSplitP) {
              ldmatrix_x4(pl + nt * 8 * kPStride + kk * 64, b[0], b[1], b[2], b[3]);
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int c = 0; c < kMT; ++c)
                  mma_16816(blk[nt][c], a[i][c][0], a[i][c][1], a[i][c][2], a[i][c][3], b[2 * i], b[2 * i + 1]);
            }
          }
        }
      } else {
        ring_values<kD, kNT, kBf16>(sm, p, st, st1, tail, pos0, warp, lane, limit_of, n0, ph, pl, blk);
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_u32(&sm.empty[st]));
        if (stages == 2) mbar_arrive(smem_u32(&sm.empty[st1]));
      }
      advance();
      if (stages == 2) advance();
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int c = 0; c < kMT; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][c][e] *= alpha[nt][e & 1];
      }
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int c = 0; c < kMT; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[nt][c][e] += row_vs[nt][e & 1] * blk[nt][c][e];
    }

    if (kQShared && !nothing) {  // the slot was written by plain stores; a bulk copy may follow
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sm.q_empty[qs]));
      if (++qs == 2) qs = 0, qphase ^= 1;
    }

    // ---- end of the piece: the rows' sums over lanes and warps
    float2 sum[kNT];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      float a = l[nt][0], b = l[nt][1];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, off);
        b += __shfl_xor_sync(0xffffffffu, b, off);
      }
      sum[nt] = make_float2(a, b);
    }
    sync_consumers();  // the maxima of the last item have been read
    if (g == 0) {
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) *reinterpret_cast<float2*>(&sm.mx[warp][8 * nt + 2 * t]) = sum[nt];
    }
    sync_consumers();
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      sum[nt] = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 o = *reinterpret_cast<const float2*>(&sm.mx[w][8 * nt + 2 * t]);
        sum[nt].x += o.x;
        sum[nt].y += o.y;
      }
    }
    const bool whole = pc.begin == 0 && pc.end == s.items;
    if (whole) {
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int n = n0 + 8 * nt + 2 * t + e;
          if (n >= p.rows) continue;
          const int tok = n / p.group;
          const float L = e ? sum[nt].y : sum[nt].x;
          const float inv = (L == 0.f || tok >= s.cnt) ? 0.f : 1.f / L;
          uint16_t* out = p.o.row(pc.b, h * p.group + n - tok * p.group, tok) + 16 * kMT * warp + 2 * g;
#pragma unroll
          for (int c = 0; c < kMT; ++c) {
            const uint32_t v = inv == 0.f ? 0u : Elem<kBf16>::pack(acc[nt][c][e] * inv, acc[nt][c][2 + e] * inv);
            *reinterpret_cast<uint32_t*>(out + 16 * c) = v;
          }
        }
      sync_consumers();  // sm.mx is written again by the next piece
      continue;
    }
    // ---- a part of a unit: leave it for the CTA that finishes last
    constexpr int kPieceFloats = kRows * (2 + kD);
    const int c0 = owner(pc.unit_begin, total, n_split), c1 = owner(pc.unit_begin + s.items - 1, total, n_split);
    auto piece_of = [&](int cta) {  // a CTA's first piece is its slot 0, a later one (a unit's begin) slot 1
      const int slot = cta == c0 && split_at(c0, total, n_split) != pc.unit_begin ? 1 : 0;
      return p.partials + (int64_t(cta) * 2 + slot) * kPieceFloats;
    };
    {
      float* out = piece_of(blockIdx.x);
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 8 * nt + 2 * t + e;
          if (warp == 0 && g == 0) __stcg(reinterpret_cast<float2*>(out) + r, make_float2(m[nt][e], e ? sum[nt].y : sum[nt].x));
          float* o = out + 2 * kRows + r * kD + 16 * kMT * warp + 2 * g;
#pragma unroll
          for (int c = 0; c < kMT; ++c)
            __stcg(reinterpret_cast<float2*>(o + 16 * c), make_float2(acc[nt][c][e], acc[nt][c][2 + e]));
        }
    }
    __threadfence();
    sync_consumers();
    if (tid == 0) sm.ticket = atomicAdd(p.tickets + c0, 1);
    sync_consumers();
    if (sm.ticket != c1 - c0) continue;
    __threadfence();
    if (tid == 0) p.tickets[c0] = 0;  // ready for the next launch
    // a warp takes every fourth row, a lane kD / 32 of its columns
    constexpr int kCols = kD / 32;
    for (int r = warp; r < kRows && n0 + r < p.rows; r += kWarps) {
      float M = -INFINITY;
      for (int i = c0 + lane; i <= c1; i += 32) M = fmaxf(M, __ldcg(reinterpret_cast<const float2*>(piece_of(i)) + r).x);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
      const float ref = M == -INFINITY ? 0.f : M;
      float L = 0.f, a[kCols];
#pragma unroll
      for (int j = 0; j < kCols; ++j) a[j] = 0.f;
      for (int i0 = c0; i0 <= c1; i0 += 32) {
        float w = 0.f, part = 0.f;
        if (i0 + lane <= c1) {
          const float2 ml = __ldcg(reinterpret_cast<const float2*>(piece_of(i0 + lane)) + r);
          w = fast_exp2(ml.x - ref);
          part = ml.x == -INFINITY ? ml.y : w * ml.y;  // (a row of NaN has no maximum; its sum is NaN)
        }
        L += part;
        const int cnt = min(32, c1 - i0 + 1);
#pragma unroll 4
        for (int j = 0; j < cnt; ++j) {
          const float wj = __shfl_sync(0xffffffffu, w, j);
          const float* src = piece_of(i0 + j) + 2 * kRows + r * kD + lane * kCols;
          float v[kCols];
          if constexpr (kCols == 4) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(src));
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
          } else {
            const float2 x = __ldcg(reinterpret_cast<const float2*>(src));
            v[0] = x.x, v[1] = x.y;
          }
#pragma unroll
          for (int k = 0; k < kCols; ++k) a[k] += wj * v[k];
        }
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
      const int n = n0 + r, tok = n / p.group;
      const float inv = (L == 0.f || tok >= s.cnt) ? 0.f : 1.f / L;
      uint16_t* out = p.o.row(pc.b, h * p.group + n - tok * p.group, tok) + lane * kCols;
#pragma unroll
      for (int k = 0; k < kCols; k += 2)
        *reinterpret_cast<uint32_t*>(out + k) = inv == 0.f ? 0u : Elem<kBf16>::pack(a[k] * inv, a[k + 1] * inv);
    }
  }
}

struct Plan {
  int nt, row_tiles, n_ctas;
  size_t bytes;
};

int max_ctas() {
  const int sms = current_device().sm_count;
  return kCtasPerSm * (sms > 0 ? sms : 148);
}

// Query rows of a KV head: up to 8, 16 or 32 in a unit.
Plan plan(const nsa_kv8_cache* c, int64_t rows) {
  Plan s;
  s.nt = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
  s.row_tiles = static_cast<int>((rows + kRowTile - 1) / kRowTile);
  const int64_t most = c->batch * c->n_kv_heads * s.row_tiles * c->max_blocks;  // items
  s.n_ctas = static_cast<int>(most < max_ctas() ? most : max_ctas());
  s.bytes = size_t(s.n_ctas) * 2 * 8 * s.nt * (2 + c->head_dim) * sizeof(float);
  return s;
}

template <int kD, int kNT, bool kBf16, bool kInt8>
int launch_attend(const CUtensorMap (&maps)[4], const AttendParams& p, cudaStream_t stream) {
  using S = Smem<kD, kNT>;
  static_assert(offsetof(S, stage) == 0 && Geo<kD>::kStageBytes % 1024 == 0, "TMA destinations");
  static_assert(offsetof(S, q) % 16 == 0 && Geo<kD>::kQStride % 16 == 0, "bulk-copy destinations");
  static_assert(offsetof(S, p_hi) % 16 == 0 && offsetof(S, p_lo) % 16 == 0 && offsetof(S, mx) % 8 == 0, "vector reads");
  static_assert(kCtasPerSm * (sizeof(S) + 1024) <= 228 * 1024, "two CTAs per SM");
  auto kernel = kv8_attend_kernel<kD, kNT, kBf16, kInt8>;
  static bool attr_set[64] = {false};
  const int dev = current_device().device;
  if (dev < 0 || dev >= 64) return fail(NSA_ERR_CUDA, "no CUDA device");
  if (!attr_set[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(S)));
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    attr_set[dev] = true;
  }
  cudaError_t e = launch_kernel(kernel, dim3(p.n_ctas), dim3(kThreads), sizeof(S), stream, maps[0], maps[1], maps[2],
                                maps[3], p);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? NSA_OK : cuda_fail(e, "kv8_attend_kernel launch");
}

template <int kD, bool kBf16, bool kInt8>
int launch_nt(int nt, const CUtensorMap (&maps)[4], const AttendParams& p, cudaStream_t stream) {
  switch (nt) {
    case 1: return launch_attend<kD, 1, kBf16, kInt8>(maps, p, stream);
    case 2: return launch_attend<kD, 2, kBf16, kInt8>(maps, p, stream);
    default: return launch_attend<kD, 4, kBf16, kInt8>(maps, p, stream);
  }
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

int nsa_kv8_attend(const nsa_kv8_cache* cache, const nsa_kv8_rows* q, const nsa_kv8_rows* o, int64_t n_heads,
                   int64_t n_tokens, const int64_t* counts, int64_t window, int64_t sink, float sm_scale,
                   void* workspace, size_t workspace_bytes, int32_t* tickets, nsa_stream_t stream) {
  clear_error();
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
  if (!workspace || workspace_bytes < s.bytes)
    return fail(NSA_ERR_WORKSPACE, "workspace of %zu bytes required (got %zu)", s.bytes, workspace ? workspace_bytes : size_t(0));
  if (!aligned16(workspace)) return fail(NSA_ERR_ALIGN, "workspace must be 16-byte aligned");
  if (!tickets) return fail(NSA_ERR_WORKSPACE, "tickets must not be NULL");
  p.row_tiles = s.row_tiles;
  p.counts = counts;
  p.window = window < 0 ? -1 : static_cast<int>(window);
  p.sink = static_cast<int>(sink);
  p.scale_log2 = sm_scale * kv8::kLog2e;
  p.n_ctas = s.n_ctas;
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
  const bool bf16 = cache->dtype == 2, int8 = cache->codes == NSA_KV8_INT8;
  if (d == 128)
    return bf16 ? (int8 ? kv8::launch_nt<128, true, true>(s.nt, maps, p, stream)
                        : kv8::launch_nt<128, true, false>(s.nt, maps, p, stream))
                : (int8 ? kv8::launch_nt<128, false, true>(s.nt, maps, p, stream)
                        : kv8::launch_nt<128, false, false>(s.nt, maps, p, stream));
  return bf16 ? (int8 ? kv8::launch_nt<64, true, true>(s.nt, maps, p, stream)
                      : kv8::launch_nt<64, true, false>(s.nt, maps, p, stream))
              : (int8 ? kv8::launch_nt<64, false, true>(s.nt, maps, p, stream)
                      : kv8::launch_nt<64, false, false>(s.nt, maps, p, stream));
}

int nsa_kv8_decode_step(const nsa_kv8_cache* cache, const nsa_kv8_rows* new_k, const nsa_kv8_rows* new_v,
                        const nsa_kv8_rows* q, const nsa_kv8_rows* o, int64_t n_heads, int64_t n_tokens,
                        const int64_t* starts, const int64_t* counts, int64_t window, int64_t sink, float sm_scale,
                        void* workspace, size_t workspace_bytes, int32_t* tickets, nsa_stream_t stream) {
  const int rc = nsa_kv8_append(cache, new_k, new_v, n_tokens, starts, counts, stream);
  if (rc) return rc;
  return nsa_kv8_attend(cache, q, o, n_heads, n_tokens, counts, window, sink, sm_scale, workspace, workspace_bytes,
                        tickets, stream);
}

}  // extern "C"
