// Attention of many rows per sequence (prompts, long continuations, the shared prefix of a batch) to the quantized paged cache, on
// the tensor cores' 128-row tiles.
//
// A unit is 256 rows (new tokens x query heads of one KV head) of one sequence, two tiles of 128, against all of its keys; the key tiles
// of all units are dealt to one CTA per SM in equal runs, as in kv_attn.cu, and parts of cut units are joined the same way. Behind a shared
// prefix a unit's keys are the prefix's tiles and then its own (or, in the prefix's own pass, the prefix's alone).
//
//   S_g = Q_g . K^T        fp16 x fp16 -> fp32 in TMEM (tcgen05 kind::f16), K the codes as fp16, exactly
//   u = (s * ks_j) * c_row + e_j,  w = 2^(u - m + 3),  l += w * 2^-e_j
//   O_g += W_g . V         W fp16 from TMEM (over S), V = fp16(code * vs_j * 2^-e_j); fp32 in TMEM;  o = O / l
// m is a row's maximum of u, rounded down, when it was last set: it is set anew, and O and l scaled, only when the maximum outgrows it by 2^12, so W
// stays at most 2^15 and O is hardly ever touched between products (2,011 tokens behind 16,000: 632 us where it might outgrow it by 2^8, 618 by 2^12).
// e_j is an exponent of the key's V scale. The keys of a tile share it where their scales lie within 2^7 of one another: it is then added to m once.
// Else each has its own (as in kv_attn.cu, where the whole scale goes into the exponent), so a large V row takes no bits from others, least of
// all where it is not seen. That costs a softmax thread four more floats a key and two more operations a score: the 2,011 tokens behind 16,000
// take 870 us where every tile is such a one, 654 with one in eight or so, 610 with none. V's one rounding
// is 2^-11 of a value, as much as that of the weights. Weights below 2^-14 lose bits, 2^-25 at most: that is 2^-28 of the row's largest
// weight times the 2^7 that V scales may differ by. l holds what keys of small V scales weigh: scales of a row may differ by 2^120.
// A key with a scale that is not finite has V = 0 and a K scale that is not a number: only the rows that see it become NaN.
//
// 896 threads, one CTA per SM: warp 0 brings pages by bulk copies (codes as they lie), warp 1 issues the products, warp 2 works out the run's segments and tells
// the others, warps 4-19 are the softmax, eight
// to a row tile, 16 rows to a warp, warps 20-23 turn K codes into fp16 tiles, warps 24-27 V codes: rows of keys, 128-byte swizzle, slabs of 64 channels. A softmax
// thread takes S by 16x256b loads, a pair of columns of every eight, of two rows: it needs the scales of a quarter of the keys (with a
// row per thread every thread loads all of them, 128 keys' floats: the shared-memory return path becomes the bound).
// The same layout is K-major for K and, with the channels as the product's N, MN-major for V, so nothing is transposed.
// Shared memory: Q 2 x 32 KB | three fp16 tiles of 32 KB (K and V in turn) | three raw tiles of 16 KB. TMEM: S0 | S1 | O0 | O1.
// Bound, per step of 128 keys and 256 rows: 2,048 cycles of the tensor pipe, as many of the exponential unit, about 2,800 of shared memory (products'
// operands 1,536, conversion 768, the keys' scales 512). Measured: 4,850, as all three wait for one another; 2,011 tokens x 32 heads behind
// 16,000 take 610 us at 1,965 MHz, 0.92 PFLOP/s (0.56 of the library's bf16 product), and 670 us call behind call for a second or more, when
// the power cap holds the SMs at 1,790 MHz (0.60 of the library's product under that cap).
#include "kv_attn.cuh"

namespace rh3 {
namespace {

constexpr int TK = 128, WBM = 256, WTHREADS = 896, SLOTS = 3, RAW = 3, SEGS = 4;
constexpr int SEG_READERS = 26;   // warps that are told of a segment: two of the service, eight of the conversion, sixteen of the softmax

template <int D>
struct KvWide {
  static constexpr int Q_BYTES = 128 * D * 2;       // a tile of 128 rows, fp16
  static constexpr int T_BYTES = TK * D * 2;        // a K or V tile, fp16
  static constexpr int R_BYTES = TK * D;            // a K or V tile, codes
  static constexpr int TILES = 2 * Q_BYTES;
  static constexpr int RAWS = TILES + SLOTS * T_BYTES;
  static constexpr int TAIL = RAWS + RAW * R_BYTES;
  static constexpr int PART = WBM * D + 2 * WBM;    // floats of a partial result
  static constexpr int O_COL = 256;                 // TMEM column of O of row tile 0
};
// one unit's part of a CTA's run
struct KvWideSegment {
  int first, n, len, pos; // of the sequence
  int b, h, u;            // sequence, KV head, row tile
  int k0, k1, kt;         // tiles [k0, k1) of the unit's kt
  int cta, parts;         // CTAs cta .. cta + parts - 1 have a part of the unit
};
struct __align__(16) KvWideTail {
  float scale[RAW][2][TK];        // as loaded with a K tile: of K, of V
  float key[2][TK];               // per key of a tile, by the tile's parity: K scale (-inf: no such key),
  float value[2][TK];             // V scale * 2^-e,
  float shift[2][TK];             // and where keys have exponents of their own, e
  float down[2][TK];              // and 2^-e
  float row[2][2][2][128];        // per row of a row tile: factor c, then l; m; two units' in turn
  uint64_t raw_full[2 * RAW];     // two for a raw tile: for when it holds K, and V, each waited for by its own warps alone
  uint64_t raw_empty[RAW], full[SLOTS], empty[SLOTS], value_full[2];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2], seg_full[SEGS], seg_empty[SEGS];
  alignas(16) uint32_t top[2][4], low[2][4];  // largest and smallest V scale above 0 of a warp's keys (bits)
  float4 tile[2];                 // by the tile's parity: e, 2^-e, not 0 where all of its keys are there, not 0 where they share e
  uint32_t pages[RAW];
  uint32_t tmem_base;
  int abort_flag;
  KvWideSegment seg[SEGS];        // the run's segments in turn; k1 = 0: there are no more
  KvWideSegment join[2];
  int parts[2];
};
template <int D>
constexpr int kv_wide_smem() { return KvWide<D>::TAIL + static_cast<int>(sizeof(KvWideTail)) + 1024; }

// as descriptor make_desc_k128, for an operand whose M or N runs along the 128-byte rows: 64-channel slabs `slab` bytes apart, groups
// of 8 rows (the product's K) 1,024
__device__ __forceinline__ uint64_t make_desc_mn128(uint32_t smem_addr, uint32_t slab) {
  uint64_t d = make_desc_k128(smem_addr);
  d &= ~(static_cast<uint64_t>(0x3FFF) << 16);
  return d | static_cast<uint64_t>(slab >> 4) << 16;
}
// D[tmem] (+)= A[tmem] * B[smem] over 128 keys: eight products of 16, A 8 columns further and B 16 rows of 128 bytes for each, in a single
// instruction sequence (as mma4_*: scalar instructions between two products cost tensor-pipe time). accumulate = 0: the first overwrites D.
__device__ __forceinline__ void mma8_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      ".reg .b32 a1, a2, a3, a4, a5, a6, a7;\n\t"
      ".reg .b64 b1, b2, b3, b4, b5, b6, b7;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.eq.b32 q, 0, 0;\n\t"
      "add.u32 a1, %1, 8;\n\tadd.u32 a2, %1, 16;\n\tadd.u32 a3, %1, 24;\n\tadd.u32 a4, %1, 32;\n\t"
      "add.u32 a5, %1, 40;\n\tadd.u32 a6, %1, 48;\n\tadd.u32 a7, %1, 56;\n\t"
      "add.u64 b1, %2, 128;\n\tadd.u64 b2, %2, 256;\n\tadd.u64 b3, %2, 384;\n\tadd.u64 b4, %2, 512;\n\t"
      "add.u64 b5, %2, 640;\n\tadd.u64 b6, %2, 768;\n\tadd.u64 b7, %2, 896;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a4], b4, %3, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a5], b5, %3, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a6], b6, %3, q;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a7], b7, %3, q;\n\t"
      "}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 16 lanes x 16 columns: thread t has columns 2 (t % 4), + 1 of each eight, of lanes t / 4 (r[4b], r[4b + 1]) and t / 4 + 8 (r[4b + 2], r[4b + 3])
__device__ __forceinline__ void tmem_ld_frag2(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st_frag2(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// 16 lanes x 64 columns: thread t has column t % 4 of each four, of lanes t / 4 (r[2b]) and t / 4 + 8 (r[2b + 1])
__device__ __forceinline__ void tmem_st_frag16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ uint64_t pk2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void upk2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul_2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add_2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max_3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// two fp16, infinities as NaN
__device__ __forceinline__ uint32_t nan_of_inf(uint32_t w) {
  const __half2 h = *reinterpret_cast<const __half2*>(&w), y = __hfma2(h, __half2half2(__ushort_as_half(0)), h);
  return *reinterpret_cast<const uint32_t*>(&y);
}

// Registers: 72 a thread at launch; service 40, softmax 88, conversion 56
static_assert(128 * 40 + 512 * 88 + 256 * 56 <= WTHREADS * 72, "the shares must not exceed the pool");

constexpr float kSlack = 12.f;   // log2 of how far a row's maximum may outgrow m
constexpr int kAlike = 7;        // V scales of a tile within 2^7 of one another share an exponent: scale * 2^-e is then in [1, 2^7)
// e of a V scale above 0, from its bits: 2^(e + 6) <= scale < 2^(e + 7). Below 2^-61 it is held at -67: V's precision falls then, and below 2^-91 it is 0
// (a scale that was written is at least 2^-40).
__device__ __forceinline__ int value_exponent(uint32_t bits) { return max(-67, static_cast<int>(bits >> 23) - 133); }

// after an abandoned wait: copies that are still on their way land before the CTA gives its shared memory back
__device__ __forceinline__ void kv_wide_settle() {
  for (int i = 0; i < 64; ++i) __nanosleep(1000);
}

// How the work is dealt. A unit's weight is what it costs in keys: UNIT_COST for Q, the join of sums and the output, and the keys that its rows
// see, prefix tiles included, taken as linear in the number u of the row tile, w(u) = base + step * u, so that sums over units have a closed
// form. CTAs get equal runs of weight (at least a tile); inside a unit weight position y stands for tile min(kt, ceil((y - UNIT_COST) / TK)),
// the last one for kt, so neighbouring runs meet at the same tile. Tiles behind the last visible key are no work and in nobody's run.
constexpr int UNIT_COST = KV_WIDE_UNIT_COST;
struct KvWideSeq {
  int first, n, len, pos, qt; // first row token of the call, new tokens, cached tokens, position of the first, row tiles
  int step;
  long long base, head;       // of one unit; weight of all units of a head
};
__device__ __forceinline__ KvWideSeq kv_wide_seq(const KvAttnParams& p, int b) {
  const KvSeq q = kv_seq<WBM, TK>(p.r, p.c.page_log2, p.group, b);
  KvWideSeq s;
  s.first = q.first, s.n = q.n, s.len = q.len, s.pos = q.pos, s.qt = q.qt;
  s.step = p.causal ? WBM / p.group : 0;
  s.base = UNIT_COST + p.r.pre_tiles * TK + max(1, p.causal ? q.pos + max(1, s.step) : q.len);
  s.head = s.base * s.qt + static_cast<long long>(s.step) * s.qt * (s.qt - 1) / 2;
  return s;
}
// tiles that row tile u works on (one at least: rows without a key are written too)
__device__ __forceinline__ int kv_wide_tiles(const KvAttnParams& p, const KvWideSeq& s, int u) {
  int seen = s.len;
  if (p.causal) seen = max(0, min(s.len, s.pos + (min((u + 1) * WBM, s.n * p.group) - 1) / p.group + 1));
  return max(1, p.r.pre_tiles + (seen + TK - 1) / TK);
}
struct KvWideWalk {
  long long x, x1, run, xb;   // position, end and length of the CTA's run; where sequence b begins
  int b;
  KvWideSeq s;
  // Every warp scans the sequences by itself.
  __device__ __forceinline__ KvWideWalk(const KvAttnParams& p) {
    const int lane = threadIdx.x & 31, per = (p.r.B + 31) >> 5;
    const int b0 = min(p.r.B, lane * per), b1 = min(p.r.B, b0 + per);
    long long own = 0;
    bool bad = false;
    for (int i = b0; i < b1; ++i) {
      own += p.c.heads * kv_wide_seq(p, i).head;
      bad |= kv_descends(p.r, i);
    }
    if (__any_sync(0xffffffffu, bad)) {   // as kv_find_run
      own = 0;
      if (lane == 0) kv_report(p.status, ST_KV_BAD_STARTS);
    }
    long long incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const long long W = __shfl_sync(0xffffffffu, incl, 31);
    run = max(static_cast<long long>(TK), (W + gridDim.x - 1) / gridDim.x);
    x = min(W, run * blockIdx.x), x1 = min(W, x + run);
    long long at = incl - own;
    int i = b0;
    const bool mine = x < x1 && at <= x && x < incl;
    if (mine) {
      for (; i < b1; ++i) {
        const long long w = p.c.heads * kv_wide_seq(p, i).head;
        if (x < at + w) break;
        at += w;
      }
    }
    const uint32_t who = __ballot_sync(0xffffffffu, mine);
    b = __shfl_sync(0xffffffffu, i, who ? __ffs(who) - 1 : 0);
    xb = __shfl_sync(0xffffffffu, at, who ? __ffs(who) - 1 : 0);
    if (x < x1) s = kv_wide_seq(p, b);
  }
  // the next unit of which the run has tiles
  __device__ __forceinline__ bool next(const KvAttnParams& p, KvWideSegment& g) {
    while (x < x1) {
      while (x - xb >= p.c.heads * s.head) {
        if (b + 1 >= p.r.B) return false;
        xb += p.c.heads * s.head;
        s = kv_wide_seq(p, ++b);
      }
      const int h = static_cast<int>((x - xb) / s.head);
      const long long xh = xb + h * s.head;   // where the head begins
      // the row tile: the last u whose units before it weigh no more than x - xh
      auto before = [&](long long u) { return s.base * u + s.step * (u * (u - 1) / 2); };
      int u = 0;
      for (int d = 1 << (31 - __clz(s.qt)); d; d >>= 1)
        if (u + d < s.qt && before(u + d) <= x - xh) u += d;
      const long long xu = xh + before(u), w = s.base + static_cast<long long>(s.step) * u;
      const int kt = kv_wide_tiles(p, s, u);
      auto tile = [&](long long y) { return y >= w ? kt : y <= UNIT_COST ? 0 : static_cast<int>(min(static_cast<long long>(kt), (y - UNIT_COST + TK - 1) / TK)); };
      const long long end = min(w, x1 - xu);
      g.k0 = tile(x - xu), g.k1 = tile(end);
      x = xu + end;
      if (g.k0 >= g.k1) continue;
      g.first = s.first, g.n = s.n, g.len = s.len, g.pos = s.pos, g.b = b, g.h = h, g.u = u, g.kt = kt;
      const long long full = min(w, static_cast<long long>(UNIT_COST) + static_cast<long long>(kt - 1) * TK + 1);   // from here on all tiles are dealt
      g.cta = static_cast<int>((xu + UNIT_COST) / run);
      g.parts = static_cast<int>((xu + full - 1) / run) - g.cta + 1;
      return true;
    }
    return false;
  }
};
__device__ __forceinline__ int kv_wide_row_tiles(const KvAttnParams& p, const KvWideSegment& g) { return g.n * p.group - g.u * WBM > 128 ? 2 : 1; }
// where the keys of tile kt are
struct KvTile {
  const int* table;   // pages
  int kt, len;        // tile and tokens of that table
};
__device__ __forceinline__ KvTile kv_wide_tile(const KvAttnParams& p, const KvWideSegment& g, int kt) {
  if (kt < p.r.pre_tiles) return KvTile{p.pre_table, kt, p.pre_len};
  return KvTile{p.r.table + g.b * p.r.table_stride, kt - p.r.pre_tiles, g.len};
}

template <int D, int FMT, bool PREFIX>
__global__ void __launch_bounds__(WTHREADS, 1) kv_wide_kernel(const KvAttnParams p) {
  using L = KvWide<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  KvWideTail* tail = reinterpret_cast<KvWideTail*>(smem + L::TAIL);
  volatile int* abort_flag = &tail->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < RAW; ++i) mbar_init(&tail->raw_empty[i], 4);
    for (int i = 0; i < 2 * RAW; ++i) mbar_init(&tail->raw_full[i], 1);
    for (int i = 0; i < SLOTS; ++i) mbar_init(&tail->full[i], 4), mbar_init(&tail->empty[i], 1);
    for (int g = 0; g < 2; ++g) {
      mbar_init(&tail->q_full[g], 1);
      mbar_init(&tail->s_full[g], 1);
      mbar_init(&tail->p_full[g], 8);
      mbar_init(&tail->o_full[g], 1);
      mbar_init(&tail->value_full[g], 4);
      tail->parts[g] = 0;
    }
    for (int i = 0; i < SEGS; ++i) mbar_init(&tail->seg_full[i], 1), mbar_init(&tail->seg_empty[i], SEG_READERS);
    tail->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&tail->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dependency_begin();
  const uint32_t tmem_base = tail->tmem_base;
  auto all_ok = [](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
  // the i-th segment of the run, once it is known; done with it
  auto segment = [&](unsigned i, bool& ok) {
    ok = all_ok(mbar_wait(&tail->seg_full[i % SEGS], i / SEGS & 1, abort_flag, p.status, ST_TIMEOUT_TMA_FULL));
    return ok && tail->seg[i % SEGS].k1 > 0;
  };
  auto release = [&](unsigned i) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&tail->seg_empty[i % SEGS]);
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
      // ------------------------------ producer: raw tiles K, V, K, V ... ------------------------------
      const int page = 1 << p.c.page_log2, tile_pages = TK >> p.c.page_log2;
      unsigned i = 0;
      bool ok = true;
      for (unsigned seg = 0; ok && segment(seg, ok); ++seg) {
        const KvWideSegment g = tail->seg[seg % SEGS];
        release(seg);
        for (int kt = g.k0; kt < g.k1 && ok; ++kt) {
          const KvTile t = kv_wide_tile(p, g, kt);
          const int at = t.kt * tile_pages + lane;
          const bool need = lane < tile_pages && (static_cast<int64_t>(at) << p.c.page_log2) < t.len;
          const int id = need ? t.table[at] : -1;
          const bool good = need && id >= 0 && id < p.c.pages;
          if (need && !good) kv_report(p.status, ST_KV_BAD_PAGE);
          const uint32_t mask = __ballot_sync(0xffffffffu, good);
          const int64_t row = (static_cast<int64_t>(id) * p.c.heads + g.h) << p.c.page_log2;
#pragma unroll 1
          for (int v = 0; v < 2; ++v, ++i) {
            const int s = i % RAW;
            ok = all_ok(mbar_wait_relaxed(&tail->raw_empty[s], (i / RAW & 1) ^ 1, abort_flag, p.status, ST_TIMEOUT_STAGE_EMPTY, 64));
            if (!ok) break;
            uint64_t* full = &tail->raw_full[i % (2 * RAW)];
            if (lane == 0) {
              tail->pages[s] = mask;
              if (mask) mbar_arrive_expect_tx(full, static_cast<uint32_t>(__popc(mask)) * page * (v ? D : D + 8));
              else mbar_arrive(full);
            }
            __syncwarp();
            if (good) {
              bulk_load(smem + L::RAWS + s * L::R_BYTES + lane * page * D, (v ? p.c.v : p.c.k) + row * D, page * D, full);
              if (!v) {
                bulk_load(&tail->scale[s][0][lane * page], p.c.ks + row, page * 4, full);
                bulk_load(&tail->scale[s][1][lane * page], p.c.vs + row, page * 4, full);
              }
            }
            __syncwarp();
          }
        }
      }
    } else if (warp == 1) {
      // ------------------------------ products ------------------------------
      // The whole warp runs the loop converged; one elected lane issues.
      constexpr uint32_t idesc_qk = make_idesc(1, 0, 0, 128, TK);
      constexpr uint32_t idesc_pv = make_idesc(1, 0, 0, 128, D) | (1u << 16);   // B runs along N
      unsigned i = 0, nq[2] = {0, 0}, np[2] = {0, 0};   // tiles taken; uses of q_full and p_full
      bool ok = true;
      auto wait_tile = [&](unsigned t) {
        return all_ok(mbar_wait_relaxed(&tail->full[t % SLOTS], t / SLOTS & 1, abort_flag, p.status, ST_TIMEOUT_TMA_FULL, 32));
      };
      auto issue_qk = [&](int r, unsigned t, bool free_tile) {
        const uint64_t q = make_desc_k128(smem_u32(smem + r * L::Q_BYTES)), k = make_desc_k128(smem_u32(smem + L::TILES + t % SLOTS * L::T_BYTES));
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < D / 64; ++c)   // slabs of 64 channels, 16 KB apart
            mma4_f16_ss(tmem_base + r * 128, q + c * (128 * 128 >> 4), k + c * (TK * 128 >> 4), idesc_qk, c);
          mma_commit(&tail->s_full[r]);
          if (free_tile) mma_commit(&tail->empty[t % SLOTS]);
        }
        __syncwarp();
      };
      for (unsigned seg = 0; ok && segment(seg, ok); ++seg) {
        const KvWideSegment& g = tail->seg[seg % SEGS];
        const int tiles = kv_wide_row_tiles(p, g), n = g.k1 - g.k0;
        release(seg);
        for (int r = 0; r < tiles && ok; ++r) {
          ok = all_ok(mbar_wait_relaxed(&tail->q_full[r], nq[r]++ & 1, abort_flag, p.status, ST_TIMEOUT_TMA_FULL, 32));
          if (ok && r == 0) ok = wait_tile(i);
          if (!ok) break;
          tc_fence_after();
          issue_qk(r, i, r == tiles - 1);
        }
        for (int j = 0; j < n && ok; ++j, i += 2) {   // i: K of tile j, i + 1: V of it, i + 2: K of the next
          for (int r = 0; r < tiles; ++r) {
            if (r == 0) ok = wait_tile(i + 1);
            ok = ok && all_ok(mbar_wait_relaxed(&tail->p_full[r], np[r]++ & 1, abort_flag, p.status, ST_TIMEOUT_P_READY, 32));
            if (!ok) break;
            tc_fence_after();
            const uint64_t v = make_desc_mn128(smem_u32(smem + L::TILES + (i + 1) % SLOTS * L::T_BYTES), TK * 128);
            if (elect_one()) {
              mma8_f16_ts(tmem_base + L::O_COL + r * D, tmem_base + r * 128, v, idesc_pv, j > 0);
              if (r == tiles - 1) mma_commit(&tail->empty[(i + 1) % SLOTS]);
              if (j == n - 1) mma_commit(&tail->o_full[r]);
            }
            __syncwarp();
            if (j + 1 < n) {
              if (r == 0) ok = wait_tile(i + 2);
              if (!ok) break;
              tc_fence_after();
              issue_qk(r, i + 2, r == tiles - 1);
            }
          }
        }
      }
    } else if (warp == 2) {
      // ------------------------------ the run ------------------------------
      KvWideWalk walk(p);
      unsigned i = 0;
      bool ok = true;
      for (bool more = true; more; ++i) {
        KvWideSegment g;
        more = walk.next(p, g);
        if (!more) g.k1 = 0;
        ok = all_ok(mbar_wait_relaxed(&tail->seg_empty[i % SEGS], (i / SEGS & 1) ^ 1, abort_flag, p.status, ST_TIMEOUT_STAGE_EMPTY, 64));
        if (!ok) break;
        if (lane == 0) {
          tail->seg[i % SEGS] = g;
          mbar_arrive(&tail->seg_full[i % SEGS]);
        }
        __syncwarp();
      }
    }
  } else if (warp >= 20) {
    // ============================ conversion: codes -> fp16 tiles ============================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    const int v = warp >= 24, tid = (threadIdx.x - 640) & 127;   // K or V
    constexpr int PER_ROW = D / 16, ROWS = 128 / PER_ROW;   // 16-code chunks of a row, rows of a round of all 128 threads
    const int q = tid % PER_ROW, r0 = tid / PER_ROW;
    const int swap = (q / 4) & 1;   // the two slabs' rows begin in the same banks: one writes its chunks in the other order
    const int chunk = (q % 4) * 2;
    // ROWS is a multiple of 8: a thread writes the same chunks of all of its rows
    const int first = (q / 4) * TK * 128 + r0 * 128 + (((chunk + swap) ^ (r0 & 7)) << 4);
    const int second = (q / 4) * TK * 128 + r0 * 128 + (((chunk + 1 - swap) ^ (r0 & 7)) << 4);
    unsigned i = v, tiles = 0;   // tile of the rings, tiles
    bool ok = true;
    for (unsigned seg = 0;; ++seg) {
      const bool more = segment(seg, ok);
      if (v ? !ok : bar_sync_or(5, 128, !ok)) break;   // the K warps leave together: they have barriers
      if (!more) break;
      const KvWideSegment g = tail->seg[seg % SEGS];
      release(seg);
      for (int kt = g.k0; kt < g.k1; ++kt, i += 2, ++tiles) {
        const KvTile t = kv_wide_tile(p, g, kt);
        const int parity = tiles & 1;
        const int s = i % RAW;
        ok = all_ok(mbar_wait(&tail->raw_full[i % (2 * RAW)], i / (2 * RAW) & 1, abort_flag, p.status, ST_TIMEOUT_TMA_FULL) &&
                    mbar_wait(&tail->empty[i % SLOTS], (i / SLOTS & 1) ^ 1, abort_flag, p.status, ST_TIMEOUT_STAGE_EMPTY));
        if (!ok && v) break;
        const uint32_t pages = tail->pages[s];
        const bool whole = pages == (0xffffffffu >> (32 - (TK >> p.c.page_log2))) && t.kt * TK + TK <= t.len;
        auto there = [&](int key) { return whole || (t.kt * TK + key < t.len && ((pages >> (key >> p.c.page_log2)) & 1u)); };
        if (v) {
          ok = all_ok(mbar_wait(&tail->value_full[parity], tiles >> 1 & 1, abort_flag, p.status, ST_TIMEOUT_TMA_FULL));
          if (!ok) break;
        } else {   // the keys' scales
          const bool is = there(tid);
          float ks = tail->scale[s][0][tid], vs = is ? tail->scale[s][1][tid] : 0.f;
          if (!(max_nan(ks, vs) < INFINITY)) vs = 0.f, ks = kNan;
          if (!(vs > 0.f)) vs = 0.f;
          const uint32_t bits = __float_as_uint(vs), most = __reduce_max_sync(0xffffffffu, bits), least = __reduce_min_sync(0xffffffffu, vs > 0.f ? bits : 0x7F7FFFFFu);
          if (lane == 0) tail->top[parity][warp & 3] = most, tail->low[parity][warp & 3] = least;
          if (bar_sync_or(5, 128, !ok)) {
            ok = false;
            break;
          }
          const uint4 top = *reinterpret_cast<const uint4*>(tail->top[parity]), low = *reinterpret_cast<const uint4*>(tail->low[parity]);
          const int e_top = value_exponent(max(max(top.x, top.y), max(top.z, top.w))), e_low = value_exponent(min(min(low.x, low.y), min(low.z, low.w)));
          const bool alike = e_top - e_low < kAlike;
          const int e = alike ? e_top : value_exponent(bits);
          const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
          tail->key[parity][tid] = is ? ks : -INFINITY;
          tail->value[parity][tid] = vs * down;
          const float shift = static_cast<float>(e);
          if (!alike) tail->shift[parity][tid] = shift, tail->down[parity][tid] = down;
          if (tid == 0) tail->tile[parity] = make_float4(shift, down, whole, alike);
          __syncwarp();
          if (lane == 0) mbar_arrive(&tail->value_full[parity]);
        }
        const uint8_t* raw = smem + L::RAWS + s * L::R_BYTES + r0 * D + q * 16;
        uint8_t* out = smem + L::TILES + i % SLOTS * L::T_BYTES;
        constexpr int N = TK / ROWS, STEP = 4;
#pragma unroll 1
        for (int k0 = 0; k0 < N; k0 += STEP) {
          uint4 w[STEP];
#pragma unroll
          for (int k = 0; k < STEP; ++k) w[k] = *reinterpret_cast<const uint4*>(raw + (k0 + k) * ROWS * D);
          if (!whole) {   // what was not loaded, or lies behind the end, may be anything: a NaN code times a weight of 0 is a NaN
#pragma unroll
            for (int k = 0; k < STEP; ++k)
              if (!there(r0 + (k0 + k) * ROWS)) w[k] = make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int k = 0; k < STEP; ++k) {
            uint32_t h[8];
            kv_codes_to_half<FMT>(swap ? w[k].z : w[k].x, h[0], h[1]);
            kv_codes_to_half<FMT>(swap ? w[k].w : w[k].y, h[2], h[3]);
            kv_codes_to_half<FMT>(swap ? w[k].x : w[k].z, h[4], h[5]);
            kv_codes_to_half<FMT>(swap ? w[k].y : w[k].w, h[6], h[7]);
            if (v) {   // times the key's scale in two fp16 pieces: rounded once
              const float f = tail->value[parity][r0 + (k0 + k) * ROWS];
              const __half hi = __float2half_rn(f), lo = __float2half_rn(f - __half2float(hi));
              const __half2 hi2 = __half2half2(hi), lo2 = __half2half2(lo);
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const __half2 c = *reinterpret_cast<const __half2*>(&h[x]);
                const __half2 y = __hfma2(c, hi2, __hmul2(c, lo2));
                h[x] = *reinterpret_cast<const uint32_t*>(&y);
              }
            }
            *reinterpret_cast<uint4*>(out + first + (k0 + k) * ROWS * 128) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(out + second + (k0 + k) * ROWS * 128) = make_uint4(h[4], h[5], h[6], h[7]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&tail->full[i % SLOTS]);
          mbar_arrive(&tail->raw_empty[s]);
        }
      }
    }
  } else {
    // ============================ softmax ============================
    // Q is brought in, and O given out, by two threads per row, half of the channels each; of S a warp has 16 rows of its TMEM quadrant,
    // a thread rows 8k + lane / 4 of these, k = 0, 1, and the column pairs 2 (lane % 4) of each eight.
    asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");
    const int rt = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t quad_off = static_cast<uint32_t>(quad * 32) << 16, half_off = static_cast<uint32_t>(half * 16) << 16;
    const uint32_t s_frag = tmem_base + rt * 128 + quad_off + half_off, o_base = tmem_base + L::O_COL + rt * D + quad_off;
    const int frag_row = quad * 32 + half * 16 + (lane >> 2);
    auto tile_bar = [&] { asm volatile("bar.sync %0, 256;" ::"r"(3 + rt) : "memory"); };
    unsigned ns = 0, no = 0;   // uses of s_full and o_full
    int parity = 0;
    bool ok = true;
    constexpr int LANES = D / 8, ROWS = 32 / LANES, N = 16 / ROWS;   // lanes of a row of Q, rows of a load, loads of the warp's 16 rows
    const int ch = lane % LANES, q_row = ((warp - 4) & 7) * 16 + lane / LANES;
    unsigned seg = 0;
    bool more = segment(0, ok);
    ok = !bar_sync_or(3 + rt, 256, !ok);   // the warps of a row tile leave together
    while (ok && more) {
      const KvWideSegment& g = tail->seg[seg % SEGS];
      const int n = g.k1 - g.k0;
      if (rt >= kv_wide_row_tiles(p, g)) {   // no rows for this tile
        parity ^= n & 1;
        release(seg);
        more = segment(++seg, ok);
        ok = !bar_sync_or(3 + rt, 256, !ok);
        continue;
      }
      float(*row_of)[128] = tail->row[seg & 1][rt];
      // ---- the rows of Q as fp16 into their tile, all loads in flight ----
      {
        uint4 x[N];
        const int flat = g.u * WBM + rt * 128 + q_row;
        int tok = flat / p.group, hh = flat - tok * p.group;
        const uint16_t* src = p.q + static_cast<int64_t>(g.first) * p.q_st + static_cast<int64_t>(g.h) * p.group * p.q_sh + ch * 8;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          x[k] = tok < g.n ? ld_global_16(src + tok * p.q_st + hh * p.q_sh) : make_uint4(0, 0, 0, 0);
          for (hh += ROWS; hh >= p.group; hh -= p.group) ++tok;
        }
        if (p.is_f16) {   // as it is
          if (lane < 16) row_of[0][((warp - 4) & 7) * 16 + lane] = p.sl2;
        } else {
#pragma unroll
          for (int k = 0; k < N; ++k) {
            uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
            float amax = 0.f, up, down;
#pragma unroll
            for (int y = 0; y < 4; ++y) amax = max_3(amax, fabsf(bf16_lo(w[y])), fabsf(bf16_hi(w[y])));
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            kv_row_factor(amax, up, down);
            if (ch == 0) row_of[0][q_row + k * ROWS] = fmaxf(p.sl2 * down, 0x1p-126f);   // not 0: a masked score is -inf
#pragma unroll
            for (int y = 0; y < 4; ++y) w[y] = pack_half2(bf16_lo(w[y]) * up, bf16_hi(w[y]) * up);
            x[k] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        uint8_t* dst = smem + rt * L::Q_BYTES + (ch / 8) * 128 * 128;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int r = q_row + k * ROWS;
          // x + 0 * x: an infinity becomes NaN. Its row has no softmax, also where all that it sees would be -inf.
          x[k] = make_uint4(nan_of_inf(x[k].x), nan_of_inf(x[k].y), nan_of_inf(x[k].z), nan_of_inf(x[k].w));
          *reinterpret_cast<uint4*>(dst + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = x[k];
        }
        fence_proxy_async_smem();
        tile_bar();
        if (half == 0 && quad == 0 && lane == 0) mbar_arrive(&tail->q_full[rt]);
      }
      // of the thread's two rows: factor, the last own key that is seen, maximum (of t) and sum
      const int warp_first = (g.u * WBM + rt * 128 + quad * 32 + half * 16) / p.group;   // token of the warp's first row: it sees least
      const int warp_last = p.causal ? g.pos + warp_first : g.len - 1;
      uint64_t c2[2];
      float m[2], l[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float c = row_of[0][frag_row + 8 * k];
        c2[k] = pk2(c, c);
        m[k] = -INFINITY, l[k] = 0.f;
      }
      for (int j = 0; j < n; ++j, parity ^= 1) {
        // S is there, and so are the keys' scales: the product waited for the tile they came with
        ok = all_ok(mbar_wait(&tail->s_full[rt], ns++ & 1, abort_flag, p.status, ST_TIMEOUT_ACC_FULL));
        if (!ok) break;
        tc_fence_after();
        const float* ks = &tail->key[parity][2 * (lane & 3)];
        const float4 tile = tail->tile[parity];
        const float e = tile.x;
        const int key0 = (g.k0 + j - p.r.pre_tiles) * TK;
        const bool cut = !PREFIX && p.causal && key0 >= 0 && key0 + TK - 1 > warp_last;   // the prefix is seen by all
        const bool alike = tile.w != 0.f, masked = cut || tile.z == 0.f || !alike;
        uint32_t w[32];
        uint64_t sum[2];
        float top[2];
        // One pass over the rows, 16 columns at a time: s * ks, its maximum, weights against the maximum as it was set before, their sum
        // (without V's exponent).
        auto pass = [&](auto mask, auto own) {
          uint64_t z2[2];
          float z[2];
          int last[2] = {0, 0};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            z[k] = (kWeightLog2 - kSlack) - (m[k] == -INFINITY ? 0.f : m[k]);
            if constexpr (!decltype(own)::value) z[k] += e;
            z2[k] = pk2(z[k], z[k]);
            top[k] = -INFINITY;
            sum[k] = pk2(0.f, 0.f);
            if constexpr (decltype(mask)::value)
              last[k] = cut ? g.pos + (g.u * WBM + rt * 128 + frag_row + 8 * k) / p.group - key0 - 2 * (lane & 3) : TK;
          }
          uint32_t r[2][8];
          float2 key[2][2];   // of the column pairs, fetched 16 columns ahead as S is
          auto fetch = [&](int c) {
            tmem_ld_frag2(s_frag + c * 16, r[c & 1]);
            key[c & 1][0] = *reinterpret_cast<const float2*>(ks + c * 16);
            key[c & 1][1] = *reinterpret_cast<const float2*>(ks + c * 16 + 8);
          };
          fetch(0);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            tmem_ld_wait8(r[c & 1]);
            if (c < 7) fetch(c + 1);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const int col = c * 16 + b * 8;
              const float2 a = key[c & 1][b];
              float2 shift, down;
              if constexpr (decltype(own)::value) {
                shift = *reinterpret_cast<const float2*>(&tail->shift[parity][2 * (lane & 3) + col]);
                down = *reinterpret_cast<const float2*>(&tail->down[parity][2 * (lane & 3) + col]);
              }
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const uint32_t* s = r[c & 1] + 4 * b + 2 * k;
                uint64_t x = mul_2(pk2(__uint_as_float(s[0]), __uint_as_float(s[1])), pk2(a.x, a.y));
                float u0, u1;
                upk2(x, u0, u1);
                if constexpr (decltype(mask)::value) {
                  if (a.x == -INFINITY || col > last[k]) u0 = -INFINITY;
                  if (a.y == -INFINITY || col + 1 > last[k]) u1 = -INFINITY;
                  x = pk2(u0, u1);
                }
                if constexpr (decltype(own)::value) {
                  upk2(add_2(fma_2(x, c2[k], z2[k]), pk2(shift.x, shift.y)), u0, u1);
                  top[k] = max_3(top[k], u0, u1);
                  u0 = kv_ex2(u0), u1 = kv_ex2(u1);
                  sum[k] = fma_2(pk2(u0, u1), pk2(down.x, down.y), sum[k]);
                } else {
                  top[k] = max_3(top[k], u0, u1);
                  upk2(fma_2(x, c2[k], z2[k]), u0, u1);
                  u0 = kv_ex2(u0), u1 = kv_ex2(u1);
                  sum[k] = add_2(sum[k], pk2(u0, u1));
                }
                w[(c * 2 + b) * 2 + k] = pack_half2(u0, u1);
              }
            }
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float c, same;
            upk2(c2[k], c, same);
            if constexpr (decltype(own)::value) top[k] -= z[k];
            else top[k] = fmaf(top[k], c, e);
          }
        };
        if (j == 0) {   // m to begin with: the maximum of the first 16 columns mostly within 2^12 of that of all
          uint32_t r[8];
          tmem_ld_frag2(s_frag, r);
          tmem_ld_wait8(r);
          const float2 a = *reinterpret_cast<const float2*>(ks), b = *reinterpret_cast<const float2*>(ks + 8);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float c, same;
            upk2(c2[k], c, same);
            float t = max_3(__uint_as_float(r[2 * k]) * a.x, __uint_as_float(r[2 * k + 1]) * a.y,
                            fmaxf(__uint_as_float(r[4 + 2 * k]) * b.x, __uint_as_float(r[5 + 2 * k]) * b.y)) * c;
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
            m[k] = masked || !(fabsf(t) < INFINITY) ? -INFINITY : floorf(t) + e;
          }
        }
        auto either = [&] {
          if (!masked) pass(std::false_type(), std::false_type());
          else if (alike) pass(std::true_type(), std::false_type());
          else pass(std::true_type(), std::true_type());
        };
        either();
        bool grew = false;
#pragma unroll
        for (int k = 0; k < 2; ++k) grew |= top[k] > m[k] + kSlack;
        if (__any_sync(0xffffffffu, grew)) {
          // a maximum outgrew m: m is set anew, O and l are scaled (the product before is done: its commit lies before s_full's), and the
          // weights made again
          float f[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float x = top[k];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            const bool set = x > m[k] + kSlack;
            x = floorf(x);
            f[k] = set ? kv_ex2(m[k] - x) : 1.f;
            l[k] *= f[k];
            if (set) m[k] = x;
          }
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[8];
              tmem_ld_frag2(o_base + half_off + c * 16, o);
              tmem_ld_wait8(o);
#pragma unroll
              for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f[(k >> 1) & 1]);
              tmem_st_frag2(o_base + half_off + c * 16, o);
            }
          }
          either();
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float even, odd;
          upk2(sum[k], even, odd);
          l[k] = fmaf(even + odd, alike ? tile.y : 1.f, l[k]);
        }
        tmem_st_frag16(s_frag, w);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tail->p_full[rt]);
      }
      ok = ok && all_ok(mbar_wait(&tail->o_full[rt], no++ & 1, abort_flag, p.status, ST_TIMEOUT_PV_DONE));
      if (ok) more = segment(seg + 1, ok);
      tc_fence_after();
      // ---- sums and maxima to the threads of the rows ----
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float x = l[k];
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        x += __shfl_xor_sync(0xffffffffu, x, 2);
        if ((lane & 3) == 0) row_of[0][frag_row + 8 * k] = x, row_of[1][frag_row + 8 * k] = m[k];
      }
      if (bar_sync_or(3 + rt, 256, !ok)) {
        ok = false;
        break;
      }
      if (more && lane < 16) {   // the next unit's rows of Q are in L2 by then
        const KvWideSegment& a = tail->seg[(seg + 1) % SEGS];
        const int next = a.u * WBM + rt * 128 + ((warp - 4) & 7) * 16 + lane, tok = next / p.group;
        if (tok < a.n) {
          const uint16_t* q = p.q + static_cast<int64_t>(a.first + tok) * p.q_st + (static_cast<int64_t>(a.h) * p.group + (next - tok * p.group)) * p.q_sh;
          prefetch_l2(q);
          if (D == 128) prefetch_l2(q + 64);
        }
      }
      const int flat = g.u * WBM + rt * 128 + row, tok = flat / p.group, hh = flat - tok * p.group;
      const bool there = tok < g.n;
      const int64_t t = g.first + tok, head = static_cast<int64_t>(g.h) * p.group + hh;
      const float l_row = row_of[0][row], m_row = row_of[1][row];
      const uint32_t o_row = o_base + half * (D / 2);   // this thread's half of the row's channels
      const bool part = !PREFIX && g.parts > 1;
      if (PREFIX || part) {
        // as the narrow kernel means it: weights 2^(t + log2 vs - m + 15) for the codes, their sum against vs
        const float m_out = m_row + kSlack, l_out = l_row;
        float* dst;   // of the prefix's rows; a partial result is [D / 4][256 rows] float4, so that lanes write, and a join reads, side by side
        if (PREFIX) {
          const int64_t at = (static_cast<int64_t>(blockIdx.x - g.cta) * p.c.heads + g.h) * p.r.T * p.group + flat;
          dst = p.pre_o + at * D + half * (D / 2);
          if (there && half == 0) *reinterpret_cast<float2*>(p.pre_ml + 2 * at) = make_float2(m_out, l_out);
        } else {
          float* slot = p.part + (2ll * blockIdx.x + (g.k0 > 0 ? 0 : 1)) * L::PART;
          dst = slot + (half * (D / 8) * WBM + rt * 128 + row) * 4;
          if (half == 0) slot[WBM * D + rt * 128 + row] = m_out, slot[WBM * D + WBM + rt * 128 + row] = l_out;
        }
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t v[16];
          tmem_ld16_async(o_row + c * 16, v);
          tmem_ld_wait16(v);
          if (!PREFIX) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              reinterpret_cast<uint4*>(dst)[(c * 4 + k) * WBM] = make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
          } else if (there) {
            st_global_32(dst + c * 16, make_uint4(v[0], v[1], v[2], v[3]), make_uint4(v[4], v[5], v[6], v[7]));
            st_global_32(dst + c * 16 + 8, make_uint4(v[8], v[9], v[10], v[11]), make_uint4(v[12], v[13], v[14], v[15]));
          }
        }
        if (part && warp == 4 && lane == 0) tail->join[g.k0 > 0 ? 0 : 1] = g, tail->parts[g.k0 > 0 ? 0 : 1] = g.parts;
      } else {
        const float inv = l_row == 0.f ? 0.f : __fdiv_rn(1.f, l_row);   // no key: 0
        uint16_t* dst = p.out + t * p.o_st + head * p.o_sh + half * (D / 2);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t v[16], w[8];
          tmem_ld16_async(o_row + c * 16, v);
          tmem_ld_wait16(v);
#pragma unroll
          for (int k = 0; k < 8; ++k) w[k] = kv_pack(__uint_as_float(v[2 * k]) * inv, __uint_as_float(v[2 * k + 1]) * inv, p.is_f16);
          if (there && (reinterpret_cast<uintptr_t>(dst) & 31) == 0) {
            st_global_32(dst + c * 16, make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7]));
          } else if (there) {
            *reinterpret_cast<uint4*>(dst + c * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(dst + c * 16 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
          }
        }
      }
      tc_fence_before();   // O has been read: the next unit's products may write it behind the next p_full
      release(seg++);
    }
    // ---- the run is done: its parts are counted, and units whose last parts they are joined, a row per thread ----
    if (!PREFIX) {
      __threadfence();
      if (!bar_sync_or(1, 512, !ok)) {
        const int tid = threadIdx.x - 128;
        if (tid < 2 && tail->parts[tid]) {
          const int first = tail->join[tid].cta;
          if (atomicAdd(p.count + first, 1) == tail->parts[tid] - 1) p.count[first] = 0;   // nobody else comes
          else tail->parts[tid] = 0;
          __threadfence();
        }
        asm volatile("bar.sync 2, 512;" ::: "memory");
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
          const int parts = tail->parts[k], first = tail->join[k].cta;
          if (!parts) continue;
          const KvWideSegment& u = tail->join[k];
          const int row = tid & 255, half = tid >> 8;
          const int flat = u.u * WBM + row, tok = flat / p.group, hh = flat - tok * p.group;
          if (tok >= u.n) continue;
          const int at = WBM * D + row;
          float m = -INFINITY, l = 0.f;
          for (int i2 = 0; i2 < parts; ++i2) m = fmaxf(m, __ldcg(p.part + kv_slot(first, i2) * L::PART + at));
          if (m == -INFINITY) m = 0.f;
          for (int i2 = 0; i2 < parts; ++i2) {
            const float* slot = p.part + kv_slot(first, i2) * L::PART + at;
            l = fmaf(__ldcg(slot + WBM), kv_ex2(__ldcg(slot) - m), l);
          }
          const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
          uint16_t* dst = p.out + (u.first + static_cast<int64_t>(tok)) * p.o_st + (static_cast<int64_t>(u.h) * p.group + hh) * p.o_sh;
#pragma unroll 1
          for (int c = half * (D / 64); c < (half + 1) * (D / 64); ++c) {
            float o[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
#pragma unroll 1
            for (int i2 = 0; i2 < parts; ++i2) {
              const float* slot = p.part + kv_slot(first, i2) * L::PART;
              const float f = kv_ex2(__ldcg(slot + at) - m);
              float4 x[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = __ldcg(reinterpret_cast<const float4*>(slot) + (c * 8 + e) * WBM + row);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                o[4 * e] = fmaf(x[e].x, f, o[4 * e]), o[4 * e + 1] = fmaf(x[e].y, f, o[4 * e + 1]);
                o[4 * e + 2] = fmaf(x[e].z, f, o[4 * e + 2]), o[4 * e + 3] = fmaf(x[e].w, f, o[4 * e + 3]);
              }
            }
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint32_t w[4];
#pragma unroll
              for (int y = 0; y < 4; ++y) w[y] = kv_pack(o[e + 2 * y] * inv, o[e + 2 * y + 1] * inv, p.is_f16);
              *reinterpret_cast<uint4*>(dst + c * 32 + e) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
      }
    }
  }

  // ------------------------------ teardown ------------------------------
  __syncwarp();
  if (*abort_flag && threadIdx.x == 0) kv_wide_settle();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int D, int FMT, bool PREFIX>
int kv_wide_start(const KvAttnParams& p, int64_t grid, cudaStream_t stream) {
  auto kern = kv_wide_kernel<D, FMT, PREFIX>;
  static std::atomic<uint64_t> allowed{0};
  if (int e = kv_allow_smem(kern, kv_wide_smem<D>(), allowed)) return e;
  return check_cuda(launch_chained(kern, dim3(static_cast<unsigned>(grid)), WTHREADS, kv_wide_smem<D>(), stream, 1, p), "kv_attn (wide) launch");
}

}  // namespace

int64_t kv_wide_part_floats(int64_t D) { return D == 128 ? KvWide<128>::PART : KvWide<64>::PART; }

int kv_wide_launch(const KvAttnParams& p, int64_t D, int kind, bool prefix, int64_t grid, cudaStream_t stream) {
  auto by_mode = [&](auto d, auto f) {
    constexpr int DD = decltype(d)::value, F = decltype(f)::value;
    return prefix ? kv_wide_start<DD, F, true>(p, grid, stream) : kv_wide_start<DD, F, false>(p, grid, stream);
  };
  using I8 = std::integral_constant<int, RH3_KIND_I8>;
  using F8 = std::integral_constant<int, RH3_KIND_F8>;
  if (D == 128) return kind == RH3_KIND_I8 ? by_mode(std::integral_constant<int, 128>(), I8()) : by_mode(std::integral_constant<int, 128>(), F8());
  return kind == RH3_KIND_I8 ? by_mode(std::integral_constant<int, 64>(), I8()) : by_mode(std::integral_constant<int, 64>(), F8());
}

}  // namespace rh3
