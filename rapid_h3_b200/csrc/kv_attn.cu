// Attention of few rows per sequence (decoding, short continuations) to the quantized paged cache.
//
// A unit is BM = 8 or 16 rows (new tokens x query heads of one KV head) of one sequence against all of its keys. What bounds it is
// reading the cache once: 2 * (D + 4) bytes per key and head. The key tiles of all units are dealt to the CTAs in equal runs
// (kv_cache.cuh), so ragged batches, single sequences and many heads all spread over the chip; of a unit that runs cut, every CTA
// leaves a partial result, and the one whose is the last joins them, in a fixed order.
//
// One CTA = a producer warp and four warps that compute, each on 32 of a tile's 128 keys with its own running maximum, sums and
// output, joined at the unit's end: no barrier among them per tile. Keys of a shared prefix come before a unit's own, or have been worked on in a pass
// before, whose parts a unit takes in (kv_plan). The producer brings pages by TMA into a ring
// (128-byte swizzle over the codes as they lie, so that the accesses below hit 32 banks), their scales by bulk copies.
//
// Products are mma.sync m16n8k16 on fp16 with the KEYS (and then the channels) as the 16 rows and the query rows as the 8 columns:
//     S^T = K . Q^T,   O^T = V^T . W^T
// so that 8 query rows fill an instruction (a 128-row tensor-core tile would be nearly empty), half of the softmax values, output registers and
// products that 16 rows take. W^T comes from S^T by movmatrix. What is left is mostly the conversion of the codes, 3 to 6
// instructions for four of them. K codes enter as code + 128 in the low bits of an fp16 (a subnormal number, (code + 128) * 2^-24,
// exact): the accumulators begin at -128 * 2^-24 * sum q, the same for every key of a row. V codes are brought to fp16 proper: there the
// offset would be summed over all keys.
// Measured, CUDA events around 50 calls: a token of each of 48 sequences of 8,192 to 16,384 tokens, 8 KV heads of 8: 203 us, 6.2 TB/s of codes and scales
// (0.94 of a copy; 217 us in a row of 2,000 calls); of up to 4,096: 53 us, 52 replayed from a graph.
// The order of channels and keys inside an mma is free, so each lane takes the channels and keys whose bytes it can load
// 16 at a time: channel order (K) 16c .. 16c+15 of lane c, key order n -> (n >> 1) | ((n & 1) << 2), output channels of
// lane group g 16g' .. 16g'+15.
#include <algorithm>

#include "kv_attn.cuh"
#include "rapidh3_b200.h"

namespace rh3 {
namespace {

constexpr int TK = 128;                 // keys of a tile
constexpr int KV_WARPS = 4;             // computing warps
// What it takes to begin and end a unit, in tiles; with the parts of a prefix pass taken in. (us with 0 / 0, 1 / 3, 2 / 3: 48 ragged sequences of up to
// 4,096 tokens 56.1, 53.8, 52.3; 64 of up to 700 behind a prefix 103, 88.2, 88.0.) 0 where every tile can have a CTA of its own.
constexpr int KV_PLAIN_COST = 2, KV_OWN_COST = 3;
constexpr int KV_NT = KV_WARPS * 32 + 32;
// no prefix; the prefix's own pass; the pass behind it, which takes its parts in; the prefix's tiles before every unit's own, in one pass
enum { MODE_PLAIN = 0, MODE_PREFIX = 1, MODE_OWN = 2, MODE_ONE = 3 };

template <int D, int NT>
struct KvNarrow {
  static constexpr int BM = 8 * NT;
  static constexpr int CTAS = NT == 1 ? 3 : 2;                    // per SM
  static constexpr int STAGES = (D == 128 ? 1 : 2) * (NT == 1 ? 2 : 3);
  static constexpr int STAGE_BYTES = 2 * TK * D;
  static constexpr int SCALES = STAGES * STAGE_BYTES;             // [STAGES][2][TK] floats
  static constexpr int TAIL = SCALES + STAGES * 2 * TK * 4;
  static constexpr int PART = BM * D + 2 * BM;                    // floats of a partial result: NT * D / 16 fragments, m, l
  static constexpr int PER = NT * (D / 16) / KV_WARPS;            // fragments that a warp joins
  static constexpr int CARRY = STAGE_BYTES / (BM * D * 4);        // parts of the prefix pass that a stage takes
  static constexpr int CARRY_ML = (BM + 2) * 2;                   // floats of a part's m and l, from an even row on
};
struct KvJoin {   // a cut unit that the CTA has a part of; parts = 0: none, or not to be joined here
  KvSegment g;
  int first, parts;
};
struct __align__(8) KvTail {
  uint64_t full[6], empty[6], parts;
  float ml[2][KV_WARPS][2][16];   // two units' (m, l) of each warp's rows in turn
  uint32_t pages[6];   // which of a stage's pages were there
  int abort_flag;
  KvJoin join[2];
};
template <int D, int NT>
constexpr int kv_narrow_smem() { return KvNarrow<D, NT>::TAIL + static_cast<int>(sizeof(KvTail)) + 1024; }

__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of fp16, one row's pair per lane, transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Four K codes of a word as fp16 pairs: int8 as (code + 128) * 2^-24, e4m3 as they are.
template <int FMT>
__device__ __forceinline__ void k_codes_to_half(uint32_t w, uint32_t& a, uint32_t& b) {
  if constexpr (FMT == RH3_KIND_I8) {
    const uint32_t u = w ^ 0x80808080u;
    a = __byte_perm(u, 0, 0x4140);
    b = __byte_perm(u, 0, 0x4342);
  } else {
    kv_codes_to_half<FMT>(w, a, b);
  }
}

// after an abandoned wait: copies that are still on their way land before the CTA gives its shared memory back
__device__ __forceinline__ void kv_settle() {
  for (int i = 0; i < 64; ++i) __nanosleep(1000);
}

// the computing warps' barrier
__device__ __forceinline__ void kv_bar() { asm volatile("bar.sync 2, %0;" ::"n"(KV_WARPS * 32) : "memory"); }

// where 16-byte chunk `ch` of key `key` lies in a swizzled tile
template <int D>
__device__ __forceinline__ int chunk_at(int key, int ch) {
  if constexpr (D == 128) return key * 128 + ((ch ^ (key & 7)) << 4);
  const int line = key >> 1;
  return line * 128 + (((((key & 1) << 2) + ch) ^ (line & 7)) << 4);
}
// the key that column n of an 8-key block stands for, and the run of D / 8 channels that output column n stands for
template <int D>
__device__ __forceinline__ int col_perm(int n) {
  return D == 128 ? (n >> 1) | ((n & 1) << 2) : n;
}

// Rows of the call: this lane's two rows of the unit
struct KvLaneRow {
  int64_t q, o;   // element offsets of the row in q and out; q < 0: no such row
  int pos;        // last key it sees
  int flat;       // row number in the prefix pass
};
template <int BM>
__device__ __forceinline__ KvLaneRow kv_lane_row(const KvAttnParams& p, const KvSegment& g, int r) {
  KvLaneRow x;
  const int flat = g.u * BM + r;
  const int i = flat / p.group, hh = flat - i * p.group;
  const bool there = i < g.s.n;
  const int64_t t = g.s.first + i, head = static_cast<int64_t>(g.h) * p.group + hh;
  x.q = there ? t * p.q_st + head * p.q_sh : -1;
  x.o = t * p.o_st + head * p.o_sh;
  x.pos = p.causal ? g.s.pos + i : g.s.len - 1;
  x.flat = (g.s.first + i) * p.group + hh;
  return x;
}
// End of the tiles of a segment that are worked on: the ones behind the last visible key are not, but one always is (its part of the ring
// is where the warps' results meet).
template <int BM>
__device__ __forceinline__ int kv_last_tile(const KvAttnParams& p, const KvSegment& g) {
  return max(g.k0 + 1, min(g.k1, p.r.pre_tiles + (kv_visible<BM>(g.s, p.group, g.u, p.causal) + TK - 1) / TK));
}
// Joins the parts of a cut unit: slot 1 of CTA `first`, slot 0 of the ones behind it, in that order. They are
// brought into the ring (which is done with) by bulk copies, as many as it holds at a time, and every thread sums its own fragments'
// values in rolled loops: the code runs once, its instructions come from L2.
template <int D, int NT>
__device__ __forceinline__ bool kv_join_parts(const KvAttnParams& p, const KvJoin& join, uint8_t* ring, KvTail* tail, uint32_t& phase) {
  using L = KvNarrow<D, NT>;
  constexpr int BM = L::BM, MT = D / 16, ROOM = L::SCALES / (L::PART * 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, c = lane & 3;
  const int col = 8 * (warp * L::PER / MT) + 2 * c;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  float4 o[L::PER];
#pragma unroll
  for (int k = 0; k < L::PER; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int i0 = 0; i0 < join.parts; i0 += ROOM) {
    const int n = min(ROOM, join.parts - i0);
    if (warp == 0) {
      asm volatile("fence.proxy.async;" ::: "memory");   // parts were written, and the ring was read, by ordinary accesses
      if (lane == 0) mbar_arrive_expect_tx(&tail->parts, n * L::PART * 4);
      __syncwarp();
      if (lane < n) bulk_load(ring + lane * L::PART * 4, p.part + kv_slot(join.first, i0 + lane) * L::PART, L::PART * 4, &tail->parts);
    }
    const bool came = mbar_wait(&tail->parts, phase, &tail->abort_flag, p.status, ST_TIMEOUT_TMA_FULL);
    if (bar_sync_or(1, KV_WARPS * 32, !came)) {
      kv_settle();
      return false;
    }
    phase ^= 1;
    const float* part = reinterpret_cast<const float*>(ring);
    float n0 = m0, n1 = m1;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float2 pm = *reinterpret_cast<const float2*>(part + i * L::PART + BM * D + col);
      n0 = fmaxf(n0, pm.x), n1 = fmaxf(n1, pm.y);
    }
    const float z0 = n0 == -INFINITY ? 0.f : n0, z1 = n1 == -INFINITY ? 0.f : n1;
    const float f0 = kv_ex2(m0 - z0), f1 = kv_ex2(m1 - z1);
    l0 *= f0, l1 *= f1;
#pragma unroll
    for (int k = 0; k < L::PER; ++k) o[k].x *= f0, o[k].y *= f1, o[k].z *= f0, o[k].w *= f1;
    m0 = n0, m1 = n1;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float* at = part + i * L::PART;
      const float2 pm = *reinterpret_cast<const float2*>(at + BM * D + col), pl = *reinterpret_cast<const float2*>(at + BM * D + BM + col);
      const float e0 = kv_ex2(pm.x - z0), e1 = kv_ex2(pm.y - z1);
      l0 = fmaf(pl.x, e0, l0), l1 = fmaf(pl.y, e1, l1);
#pragma unroll
      for (int k = 0; k < L::PER; ++k) {
        const float4 x = reinterpret_cast<const float4*>(at)[(warp * L::PER + k) * 32 + lane];
        o[k].x = fmaf(x.x, e0, o[k].x), o[k].y = fmaf(x.y, e1, o[k].y), o[k].z = fmaf(x.z, e0, o[k].z), o[k].w = fmaf(x.w, e1, o[k].w);
      }
    }
    kv_bar();   // before the ring is written again
  }
  const float i0 = l0 == 0.f ? 0.f : __fdiv_rn(1.f, l0), i1 = l1 == 0.f ? 0.f : __fdiv_rn(1.f, l1);
  const KvLaneRow r0 = kv_lane_row<BM>(p, join.g, col), r1 = kv_lane_row<BM>(p, join.g, col + 1);
#pragma unroll
  for (int k = 0; k < L::PER; ++k) {   // a fragment is two neighbouring channels of two rows
    const int ch = D / 8 * col_perm<D>(gq) + 2 * (warp * L::PER % MT + k);
    if (r0.q >= 0) *reinterpret_cast<uint32_t*>(p.out + r0.o + ch) = kv_pack(o[k].x * i0, o[k].z * i0, p.is_f16);
    if (r1.q >= 0) *reinterpret_cast<uint32_t*>(p.out + r1.o + ch) = kv_pack(o[k].y * i1, o[k].w * i1, p.is_f16);
  }
  return true;
}

// What the prefix pass left for the rows of an own unit, which lie in one or two of its units: so many parts at most.
struct KvCarry {
  int flat, rows;         // the unit's first row in the prefix pass, its rows
  int edge, n0, n1;       // rows before `edge` have n0 parts, the others n1
};
template <int BM>
__device__ __forceinline__ KvCarry kv_carry(const KvAttnParams& p, const KvSegment& g) {
  KvCarry c;
  c.flat = g.s.first * p.group + g.u * BM;
  c.rows = min(BM, g.s.n * p.group - g.u * BM);
  const int units = (p.r.T * p.group + p.pre_bm - 1) / p.pre_bm, u = c.flat / p.pre_bm;
  auto parts = [&](int unit) {
    const int x = (g.h * units + unit) * p.pre_unit;
    return (x + p.pre_last) / p.pre_run - (x + p.pre_first) / p.pre_run + 1;
  };
  c.edge = (u + 1) * p.pre_bm - c.flat;
  c.n0 = parts(u);
  c.n1 = c.edge < c.rows ? parts(u + 1) : 0;
  return c;
}

template <int D, int FMT, int MODE, int NT>
__global__ void __launch_bounds__(KV_NT, KvNarrow<D, NT>::CTAS)
kv_attn_kernel(const __grid_constant__ CUtensorMap tma_k, const __grid_constant__ CUtensorMap tma_v, const KvAttnParams p) {
  using L = KvNarrow<D, NT>;
  constexpr int S = L::STAGES, BM = L::BM, MT = D / 16, CH = D / 8, QW = D / 4;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* scales = reinterpret_cast<float*>(smem + L::SCALES);
  KvTail* tail = reinterpret_cast<KvTail*>(smem + L::TAIL);
  volatile int* abort_flag = &tail->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&tail->full[s], 1);
      mbar_init(&tail->empty[s], KV_WARPS);
    }
    mbar_init(&tail->parts, 1);
    tail->abort_flag = 0;
    tail->join[0].parts = tail->join[1].parts = 0;
    fence_barrier_init();
  }
  __syncthreads();
  grid_dependency_begin();
  const KvRun run = kv_find_run<BM, TK>(p.r, p.c.page_log2, p.c.heads, p.group, p.cost, p.status);
  KvWalk<BM, TK> walk(run);
  KvSegment g;

  if (warp == KV_WARPS) {
    // ------------------------------ producer ------------------------------
    if (lane == 0) {
      tma_prefetch_desc(&tma_k);
      tma_prefetch_desc(&tma_v);
    }
    const int page = 1 << p.c.page_log2, tile_pages = TK >> p.c.page_log2;
    int stage = 0;
    uint32_t ph = 1;
    while (walk.next(p.r, p.c.page_log2, p.c.heads, p.group, p.cost, g)) {
      if (MODE == MODE_OWN && g.k0 == 0) {   // what the prefix pass left goes through the ring before the keys do
        const KvCarry c = kv_carry<BM>(p, g);
        const int64_t rows = static_cast<int64_t>(p.r.T) * p.group;
        const int parts = max(c.n0, c.n1);
        for (int s0 = 0; s0 < parts; s0 += L::CARRY) {
          if (!__all_sync(0xffffffffu, mbar_wait(&tail->empty[stage], ph, abort_flag, p.status, ST_TIMEOUT_STAGE_EMPTY))) {
            kv_settle();
            return;
          }
          const int n = min(L::CARRY, parts - s0);
          if (lane == 0) mbar_arrive_expect_tx(&tail->full[stage], n * (c.rows * D * 4 + L::CARRY_ML * 4));
          __syncwarp();
          if (lane < n) {
            const int64_t at = (static_cast<int64_t>(s0 + lane) * p.c.heads + g.h) * rows + c.flat;
            bulk_load(smem + stage * L::STAGE_BYTES + lane * BM * D * 4, p.pre_o + at * D, c.rows * D * 4, &tail->full[stage]);
            bulk_load(scales + stage * 2 * TK + lane * L::CARRY_ML, p.pre_ml + 2 * (at & ~1ll), L::CARRY_ML * 4, &tail->full[stage]);
          }
          __syncwarp();
          if (++stage == S) stage = 0, ph ^= 1;
        }
      }
      const int kend = kv_last_tile<BM>(p, g);
      for (int kt = g.k0; kt < kend; ++kt) {
        const bool pre = MODE == MODE_ONE && kt < p.r.pre_tiles;
        const int at = (MODE == MODE_ONE && !pre ? kt - p.r.pre_tiles : kt) * tile_pages + lane;
        const bool need = lane < tile_pages && (static_cast<int64_t>(at) << p.c.page_log2) < (pre ? p.pre_len : g.s.len);
        const int id = need ? (pre ? p.pre_table + at : p.r.table + g.b * p.r.table_stride + at)[0] : -1;
        const bool good = need && id >= 0 && id < p.c.pages;
        if (need && !good) kv_report(p.status, ST_KV_BAD_PAGE);
        const uint32_t mask = __ballot_sync(0xffffffffu, good);
        if (!__all_sync(0xffffffffu, mbar_wait(&tail->empty[stage], ph, abort_flag, p.status, ST_TIMEOUT_STAGE_EMPTY))) {
          kv_settle();
          return;
        }
        if (lane == 0) {
          tail->pages[stage] = mask;
          if (mask) mbar_arrive_expect_tx(&tail->full[stage], static_cast<uint32_t>(__popc(mask)) * page * (2 * D + 8));
          else mbar_arrive(&tail->full[stage]);
        }
        __syncwarp();
        if (good) {
          const int64_t row = (static_cast<int64_t>(id) * p.c.heads + g.h) << p.c.page_log2;
          const int y = static_cast<int>(row * D / 128);
          uint8_t* k = smem + stage * L::STAGE_BYTES + lane * page * D;
          float* sc = scales + stage * 2 * TK + lane * page;
          tma_load_2d(k, &tma_k, 0, y, &tail->full[stage]);
          tma_load_2d(k + TK * D, &tma_v, 0, y, &tail->full[stage]);
          bulk_load(sc, p.c.ks + row, page * 4, &tail->full[stage]);
          bulk_load(sc + TK, p.c.vs + row, page * 4, &tail->full[stage]);
        }
        __syncwarp();
        if (++stage == S) stage = 0, ph ^= 1;
      }
    }
    return;
  }

  // ------------------------------ computing warps ------------------------------
  // lane = (gq, c). K and V side: key gq of an 8-key block, channels of quarter c; query rows 8 nt + 2c + e are the lane's columns
  const int gq = lane >> 2, c = lane & 3;
  const int kg = col_perm<D>(gq), kc0 = col_perm<D>(2 * c), kc1 = col_perm<D>(2 * c + 1);
  const int ch0 = CH * col_perm<D>(gq);   // first of the lane's D / 8 output channels
  bool ok = true;
  int stage = 0, unit = 0;
  uint32_t ph = 0;
  while (walk.next(p.r, p.c.page_log2, p.c.heads, p.group, p.cost, g)) {
    // query rows as B fragments of D / 16 products, row 8 nt + gq, channels 16c .. 16c+15 of each 64; per column: the factor from
    // accumulator to base-2 exponent, and where the accumulator begins
    uint32_t qb[NT][D / 16][2];
    float cf[NT][2], base[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int64_t at = kv_lane_row<BM>(p, g, 8 * nt + gq).q;
      uint32_t x[QW / 2];
#pragma unroll
      for (int j = 0; j < QW / 8; ++j) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (at >= 0) v = ld_global_16(p.q + at + (j >> 1) * 64 + c * 16 + (j & 1) * 8);
        x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
      }
      float amax = 0.f, up, down;
#pragma unroll
      for (int j = 0; j < QW / 2; ++j) {
        const float2 f = kv_unpack(x[j], p.is_f16);
        amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      kv_row_factor(amax, up, down);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < QW / 2; ++j) {
        const float2 f = kv_unpack(x[j], p.is_f16);
        const __half2 h = __floats2half2_rn(f.x * up, f.y * up);
        qb[nt][j >> 1][j & 1] = *reinterpret_cast<const uint32_t*>(&h);
        const float2 r = __half22float2(h);
        sum += r.x + r.y;
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      // a row with an infinity has no softmax, also where all that it sees would be -inf (a NaN among its values does the same by itself)
      const float f = amax < INFINITY ? p.sl2 * down * (FMT == RH3_KIND_I8 ? 16777216.f : 1.f) : kNan;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        cf[nt][e] = __shfl_sync(0xffffffffu, f, (2 * c + e) * 4);
        base[nt][e] = FMT == RH3_KIND_I8 ? __shfl_sync(0xffffffffu, sum * -0x1p-17f, (2 * c + e) * 4) : 0.f;
      }
    }
    float o[NT][MT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int j = 0; j < MT; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
    }

    if (MODE == MODE_OWN && g.k0 == 0) {   // what the prefix pass left for the rows: warp w begins with parts w, w + 4, ...
      const KvCarry cr = kv_carry<BM>(p, g);
      const int64_t rows = static_cast<int64_t>(p.r.T) * p.group;
      const int parts = max(cr.n0, cr.n1);
      for (int s0 = 0; s0 < parts && ok; s0 += L::CARRY) {
        ok = __all_sync(0xffffffffu, mbar_wait(&tail->full[stage], ph, abort_flag, p.status, ST_TIMEOUT_TMA_FULL));
        if (!ok) break;
#pragma unroll 1
        for (int s = warp; s < min(L::CARRY, parts - s0); s += KV_WARPS) {
          const int odd = static_cast<int>(((static_cast<int64_t>(s0 + s) * p.c.heads + g.h) * rows + cr.flat) & 1);
          const float* part = reinterpret_cast<const float*>(smem + stage * L::STAGE_BYTES) + s * BM * D + ch0;
          const float* ml = scales + stage * 2 * TK + s * L::CARRY_ML + 2 * odd;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int r = 8 * nt + 2 * c + e;
              const bool is = r < cr.rows && s0 + s < (r < cr.edge ? cr.n0 : cr.n1);
              const float pm = is ? ml[2 * r] : -INFINITY, pl = is ? ml[2 * r + 1] : 0.f;
              const float nm = fmaxf(m[nt][e], pm);
              const float zz = nm == -INFINITY ? 0.f : nm;
              const float f = kv_ex2(m[nt][e] - zz), fp = kv_ex2(pm - zz);
              m[nt][e] = nm;
              l[nt][e] = l[nt][e] * f + (gq == 0 ? pl * fp : 0.f);   // l is a sum over the column's eight lanes
              if (is) {
#pragma unroll
                for (int j = 0; j < MT; j += 2) {
                  const float4 x = *reinterpret_cast<const float4*>(part + r * D + 2 * j);
                  o[nt][j][e] = o[nt][j][e] * f + x.x * fp;
                  o[nt][j][2 + e] = o[nt][j][2 + e] * f + x.y * fp;
                  o[nt][j + 1][e] = o[nt][j + 1][e] * f + x.z * fp;
                  o[nt][j + 1][2 + e] = o[nt][j + 1][2 + e] * f + x.w * fp;
                }
              }
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tail->empty[stage]);
        if (++stage == S) stage = 0, ph ^= 1;
      }
    }
    const int kend = kv_last_tile<BM>(p, g);
    const int pos_first = p.causal ? g.s.pos + g.u * BM / p.group : g.s.len - 1;
    for (int kt = g.k0; kt < kend && ok; ++kt) {
      if (!__all_sync(0xffffffffu, mbar_wait(&tail->full[stage], ph, abort_flag, p.status, ST_TIMEOUT_TMA_FULL))) {
        ok = false;
        break;
      }
      uint8_t* sk = smem + stage * L::STAGE_BYTES + warp * 32 * D;
      uint8_t* sv = sk + TK * D;
      const float* sks = scales + stage * 2 * TK + warp * 32;
      const uint32_t pages = tail->pages[stage];
      const bool pre = MODE == MODE_ONE && kt < p.r.pre_tiles;   // of the prefix, which every row sees
      const int tile0 = (MODE == MODE_ONE && !pre ? kt - p.r.pre_tiles : kt) * TK, len = pre ? p.pre_len : g.s.len;
      const int key0 = warp * 32, pos0 = tile0 + key0;
      const bool whole = pages == (0xffffffffu >> (32 - (TK >> p.c.page_log2))) && tile0 + TK <= len;
      const bool masked = !whole || (!pre && tile0 + TK - 1 > pos_first);
      auto there = [&](int key) { return pos0 + key < len && ((pages >> ((key0 + key) >> p.c.page_log2)) & 1u); };
      if (!whole) {
        // what was not loaded, or lies behind the sequence's end, may hold anything: a NaN code times a weight of 0 is a NaN
        if (!there(lane)) {
#pragma unroll
          for (int ch = 0; ch < D / 16; ++ch) {
            *reinterpret_cast<uint4*>(sk + chunk_at<D>(lane, ch)) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(sv + chunk_at<D>(lane, ch)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();   // before the stage is handed back to the TMA
        }
        __syncwarp();
      }
      // ---- scores: 2 blocks of 16 keys; u[nt][block][row of the block: gq, gq + 8][column] ----
      float u[NT][2][2][2];
      float iv[2][2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        uint32_t w[2][QW / 4];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int i = 0; i < D / 64; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(sk + chunk_at<D>(kb * 16 + r * 8 + kg, 4 * i + c));
            w[r][4 * i] = v.x, w[r][4 * i + 1] = v.y, w[r][4 * i + 2] = v.z, w[r][4 * i + 3] = v.w;
          }
        float acc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][2] = base[nt][0], acc[nt][1] = acc[nt][3] = base[nt][1];
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          uint32_t a[4];
          k_codes_to_half<FMT>(w[0][j], a[0], a[2]);
          k_codes_to_half<FMT>(w[1][j], a[1], a[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(acc[nt], a, qb[nt][j][0], qb[nt][j][1]);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float ks = sks[kb * 16 + r * 8 + kg];
          const float v_scale = sks[TK + kb * 16 + r * 8 + kg], vs = fmaxf(v_scale, kVsMin);
          // A row of K or V that is not finite has codes 0. fmaxf would drop a NaN of V's, and what the offset of the codes leaves of a sum
          // that should be 0 times an infinite scale may be -inf, a key left out.
          if (!(max_nan(ks, v_scale) < INFINITY)) ks = kNan;
          const float lv = kv_lg2(vs);
          iv[kb][r] = kv_rcp(vs);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            u[nt][kb][r][0] = fmaf(acc[nt][2 * r] * ks, cf[nt][0], lv);
            u[nt][kb][r][1] = fmaf(acc[nt][2 * r + 1] * ks, cf[nt][1], lv);
          }
        }
      }
      if (masked) {
        int pos[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) pos[nt][e] = kv_lane_row<BM>(p, g, 8 * nt + 2 * c + e).pos;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int key = kb * 16 + r * 8 + kg;
            const bool is = there(key);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                if (!is || (!pre && pos0 + key > pos[nt][e])) u[nt][kb][r][e] = -INFINITY;
              }
          }
      }
      // ---- running maximum ----
      float n[NT][2], z[NT][2];
      bool grew = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(fmaxf(u[nt][0][0][e], u[nt][0][1][e]), fmaxf(u[nt][1][0][e], u[nt][1][1][e]));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          n[nt][e] = fmaxf(m[nt][e], x);
          grew |= n[nt][e] > m[nt][e];
          z[nt][e] = (n[nt][e] == -INFINITY ? 0.f : n[nt][e]) - kWeightLog2;   // nothing seen yet: weights 2^-inf = 0
        }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float f0 = kv_ex2(m[nt][0] - (z[nt][0] + kWeightLog2)), f1 = kv_ex2(m[nt][1] - (z[nt][1] + kWeightLog2));
          l[nt][0] *= f0, l[nt][1] *= f1;
          m[nt][0] = n[nt][0], m[nt][1] = n[nt][1];
#pragma unroll
          for (int j = 0; j < MT; ++j) o[nt][j][0] *= f0, o[nt][j][1] *= f1, o[nt][j][2] *= f0, o[nt][j][3] *= f1;
        }
      }
      // ---- weights, as B fragments (16 keys x 8 rows) ----
      uint32_t wb[NT][2][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float w0 = kv_ex2(u[nt][kb][r][0] - z[nt][0]), w1 = kv_ex2(u[nt][kb][r][1] - z[nt][1]);
            if (!masked) {
              l[nt][0] = fmaf(w0, iv[kb][r], l[nt][0]);
              l[nt][1] = fmaf(w1, iv[kb][r], l[nt][1]);
            } else {   // a key that a row does not see may have any scale
              if (w0 != 0.f) l[nt][0] = fmaf(w0, iv[kb][r], l[nt][0]);
              if (w1 != 0.f) l[nt][1] = fmaf(w1, iv[kb][r], l[nt][1]);
            }
            wb[nt][kb][r] = transpose8(pack_half2(w0, w1));
          }
      // ---- O^T += V^T . W^T ----
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        constexpr int VW = D / 32;   // words of D / 8 channels
        uint32_t v[4][VW];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = kb * 16 + (i >> 1) * 8 + ((i & 1) ? kc1 : kc0);
          if constexpr (D == 128) {
            const uint4 x = *reinterpret_cast<const uint4*>(sv + chunk_at<D>(key, kg));
            v[i][0] = x.x, v[i][1] = x.y, v[i][2] = x.z, v[i][3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(sv + chunk_at<D>(key, gq >> 1) + (gq & 1) * 8);
            v[i][0] = x.x, v[i][1] = x.y;
          }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int b = 0; b < 2; ++b) {   // bytes 2b and 2b + 1: rows gq and gq + 8 of output block 2w + b
            const uint32_t sel = b ? 0x7362 : 0x5140;
            uint32_t a[4];
            kv_codes_to_half<FMT>(__byte_perm(v[0][w], v[1][w], sel), a[0], a[1]);
            kv_codes_to_half<FMT>(__byte_perm(v[2][w], v[3][w], sel), a[2], a[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][2 * w + b], a, wb[nt][kb][0], wb[nt][kb][1]);
          }
      }
      __syncwarp();
      if (kt + 1 == kend) break;   // the last tile's stage is kept for the join below
      if (lane == 0) mbar_arrive(&tail->empty[stage]);
      if (++stage == S) stage = 0, ph ^= 1;
    }

    // ---- join the four warps: each leaves its sums where its own keys of the last tile were ----
    float4* own = reinterpret_cast<float4*>(smem + stage * L::STAGE_BYTES + warp * 32 * D);   // fragments of nt = 0 over its K rows, 1 over V
    float(*ml)[2][16] = tail->ml[unit & 1];
    ++unit;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4);
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
        l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
        if (gq == 0) ml[warp][0][8 * nt + 2 * c + e] = m[nt][e], ml[warp][1][8 * nt + 2 * c + e] = l[nt][e];
      }
#pragma unroll
      for (int j = 0; j < MT; ++j) own[nt * (TK * D / 16) + j * 32 + lane] = make_float4(o[nt][j][0], o[nt][j][1], o[nt][j][2], o[nt][j][3]);
    }
    if (bar_sync_or(1, KV_WARPS * 32, !ok)) {
      kv_settle();
      return;
    }
    // this thread: rows col, col + 1 of fragments warp * PER + k
    const int jnt = warp * L::PER / MT, col = 8 * jnt + 2 * c;
    float M[2], sum[2] = {0.f, 0.f};
    float4 x[L::PER];
    {
      float f[KV_WARPS][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        M[e] = -INFINITY;
#pragma unroll
        for (int w = 0; w < KV_WARPS; ++w) M[e] = fmaxf(M[e], ml[w][0][col + e]);
        const float zz = M[e] == -INFINITY ? 0.f : M[e];
#pragma unroll
        for (int w = 0; w < KV_WARPS; ++w) {
          f[w][e] = kv_ex2(ml[w][0][col + e] - zz);
          sum[e] = fmaf(ml[w][1][col + e], f[w][e], sum[e]);
        }
      }
#pragma unroll
      for (int k = 0; k < L::PER; ++k) x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < KV_WARPS; ++w) {
        const float4* src = reinterpret_cast<const float4*>(smem + stage * L::STAGE_BYTES + w * 32 * D) + jnt * (TK * D / 16) + (warp * L::PER % MT) * 32 + lane;
#pragma unroll
        for (int k = 0; k < L::PER; ++k) {
          const float4 y = src[k * 32];
          x[k].x = fmaf(y.x, f[w][0], x[k].x), x[k].y = fmaf(y.y, f[w][1], x[k].y), x[k].z = fmaf(y.z, f[w][0], x[k].z), x[k].w = fmaf(y.w, f[w][1], x[k].w);
        }
      }
    }
    fence_proxy_async_smem();   // the stage goes back to the TMA
    __syncwarp();
    if (lane == 0) mbar_arrive(&tail->empty[stage]);
    if (++stage == S) stage = 0, ph ^= 1;

    if (MODE != MODE_PREFIX && (g.k0 > 0 || g.k1 < g.s.kt)) {   // a part of a unit
      const int at = g.x / run.run, parts = (g.x + g.s.kt - 1) / run.run - at + 1;
      float* slot = p.part + (2ll * blockIdx.x + (g.k0 > 0 ? 0 : 1)) * L::PART;
#pragma unroll
      for (int k = 0; k < L::PER; ++k) reinterpret_cast<float4*>(slot)[(warp * L::PER + k) * 32 + lane] = x[k];
      if (gq == 0 && warp * L::PER % MT == 0) {
        *reinterpret_cast<float2*>(slot + BM * D + col) = make_float2(M[0], M[1]);
        *reinterpret_cast<float2*>(slot + BM * D + BM + col) = make_float2(sum[0], sum[1]);
      }
      if (threadIdx.x == 0) {   // counted, and joined by whose part is the last, when the run is done
        KvJoin& join = tail->join[g.k0 > 0 ? 0 : 1];
        join.g = g, join.first = at, join.parts = parts;
      }
      continue;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const KvLaneRow r = kv_lane_row<BM>(p, g, col + e);
      if (r.q < 0) continue;
      if constexpr (MODE == MODE_PREFIX) {
        const long long at = (static_cast<long long>(blockIdx.x - g.x / run.run) * p.c.heads + g.h) * p.r.T * p.group + r.flat;
        if (gq == 0 && warp * L::PER % MT == 0) *reinterpret_cast<float2*>(p.pre_ml + 2 * at) = make_float2(M[e], sum[e]);
#pragma unroll
        for (int k = 0; k < L::PER; ++k)
          *reinterpret_cast<float2*>(p.pre_o + at * D + ch0 + 2 * (warp * L::PER % MT + k)) = e ? make_float2(x[k].y, x[k].w) : make_float2(x[k].x, x[k].z);
      } else {
        const float inv = sum[e] == 0.f ? 0.f : __fdiv_rn(1.f, sum[e]);   // no key: 0
#pragma unroll
        for (int k = 0; k < L::PER; ++k)
          *reinterpret_cast<uint32_t*>(p.out + r.o + ch0 + 2 * (warp * L::PER % MT + k)) =
              kv_pack((e ? x[k].y : x[k].x) * inv, (e ? x[k].w : x[k].z) * inv, p.is_f16);
      }
    }
  }
  if constexpr (MODE != MODE_PREFIX) {
    __threadfence();
    kv_bar();
    if (threadIdx.x < 2) {
      KvJoin& join = tail->join[threadIdx.x];
      if (join.parts) {
        if (atomicAdd(p.count + join.first, 1) == join.parts - 1) p.count[join.first] = 0;   // nobody else comes
        else join.parts = 0;
      }
      __threadfence();
    }
    kv_bar();
    uint32_t phase = 0;
#pragma unroll 1
    for (int i = 0; i < 2; ++i)
      if (tail->join[i].parts && !kv_join_parts<D, NT>(p, tail->join[i], smem, tail, phase)) return;
  }
}

int kv_maps(CUtensorMap* mk, CUtensorMap* mv, const KvCache& c, int64_t D) {
  const uint64_t page = 1ull << c.page_log2, rows = static_cast<uint64_t>(c.pages) * c.heads * page * D / 128;
  const uint32_t box = static_cast<uint32_t>(page * D / 128);
  if (int e = make_tmap_2d(mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.k, 128, rows, 128, 128, box, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
  return make_tmap_2d(mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.v, 128, rows, 128, 128, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// CTAs of a pass: as many as stay on the chip together, no more than there can be tiles
int64_t kv_grid(int64_t units, int64_t kt, int per_sm) {
  const int64_t most = static_cast<int64_t>(per_sm) * device_sm_count();
  return units * kt < most ? units * kt : most;
}

template <int D, int FMT, int MODE, int NT>
int kv_launch(const CUtensorMap& mk, const CUtensorMap& mv, const KvAttnParams& p, int64_t grid, cudaStream_t stream) {
  auto kern = kv_attn_kernel<D, FMT, MODE, NT>;
  const int smem = kv_narrow_smem<D, NT>();
  static std::atomic<uint64_t> allowed{0};
  if (int e = kv_allow_smem(kern, smem, allowed)) return e;
  return check_cuda(launch_chained(kern, dim3(static_cast<unsigned>(grid)), KV_NT, smem, stream, 1, mk, mv, p), "kv_attn launch");
}

// rh3_kv_attn_use_wide: -1 by cost, 0 never, 1 always, 2 never and a prefix has a pass of its own
std::atomic<int> g_use_wide{-1};

// The plan of a call: which kernel and rows per unit, grids and the pieces of its workspace.
struct KvPass {
  int nt;                       // narrow: units of 8 * nt rows; 0: wide, units of 256
  int64_t bm, kt, w, grid;      // rows of a unit, key tiles of a unit and weight of the pass at most, CTAs
  int cost;                     // what a unit weighs besides its tiles
};
// What a pass costs, by what it costs per SM: here 0.8 us for a tile of 16 rows and 0.5 for one of 8; in the wide kernel 10 us to begin with (tensor
// memory, Q, the first tile's latency, the output), 2.6 us for a tile of 256 rows and 1.8 for one of up to 128. Measured at 128 channels; with
// 8 KV heads 24 rows x 700 keys 17 / 23 us here / there, 512 x 12,000 130 / 40, 8,044 x 18,000 3,029 / 620. Sequences count as equally long.
struct KvCost {
  double narrow, wide;
};
KvCost kv_cost(int64_t heads, int64_t rows, int64_t seqs, int64_t kt) {
  const int64_t each = (rows + seqs - 1) / seqs;
  const double work = static_cast<double>(heads) * seqs * (kt < 1 ? 1 : kt) / device_sm_count();
  return {(rows <= 8 * seqs ? 0.5 : 0.8 * ((each + 15) / 16)) * work, 10.0 + (each > 128 ? 2.6 * ((each + 255) / 256) : 1.8) * work};
}
KvPass kv_pass(int64_t heads, int64_t rows, int64_t seqs, int64_t kt, int cost) {
  KvPass x{};
  x.cost = cost;
  x.nt = rows <= 8 * seqs ? 1 : 2;
  const int use = g_use_wide.load(std::memory_order_relaxed);
  const KvCost cost_us = kv_cost(heads, rows, seqs, kt);
  if (use >= 0) x.nt = use == 1 ? 0 : x.nt;
  else if ((rows + seqs - 1) / seqs > 16 && cost_us.wide < cost_us.narrow) x.nt = 0;
  x.bm = x.nt ? 8 * x.nt : KV_WIDE_BM;
  x.kt = kt < 1 ? 1 : kt;
  const int64_t units = heads * (rows / x.bm + seqs);
  const int per_sm = x.nt == 0 ? 1 : x.nt == 1 ? 3 : 2;
  x.grid = kv_grid(units, x.kt, per_sm);
  if (x.grid < static_cast<int64_t>(per_sm) * device_sm_count()) x.cost = 0;
  x.w = units * (x.kt + x.cost);
  return x;
}
struct KvPlan {
  KvPass own, pre;              // pre.grid = 0: no pass of its own for the prefix (none, or its tiles come before the units' own)
  bool one;                     // its tiles come before the units' own
  int64_t pre_run, pre_unit, pre_first, pre_last;   // see KvAttnParams
  int64_t pre_splits;           // into how many parts the prefix pass's units may fall
  int64_t part, pre_ml, pre_o, bytes;   // byte offsets
};
KvPlan kv_plan(int64_t heads, int64_t group, int64_t page, int64_t D, int64_t per_seq, int64_t B, int64_t T, int64_t prefix) {
  KvPlan x{};
  const int64_t rows = T * group, pre_kt = (prefix + TK - 1) / TK, own_kt = (per_seq * page + TK - 1) / TK, seqs = B < T ? B : T;
  auto take = [&](int64_t bytes) {
    const int64_t at = x.bytes;
    x.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  x.own = kv_pass(heads, rows, seqs, own_kt, prefix > 0 ? KV_OWN_COST : KV_PLAIN_COST);
  if (prefix > 0 && x.own.nt) {
    // A pass of its own for the prefix takes some 7 us besides its work (its launch, its parts written and taken in). Without it every sequence's units
    // work on the prefix's tiles, from L2 mostly. (us in one pass / in two, 8 KV heads of 4, a row per sequence: 6 sequences behind 700
    // tokens 11.8 / 15.9, 64 30.5 / 31.8; 6 behind 4,000 17.8 / 25.2, 16 30.7 / 27.7; 64 x 8 rows behind 12,000 222 / 197, with the prefix on
    // the tensor-core tiles 88.)
    const double here = kv_cost(heads, rows, seqs, pre_kt).narrow;
    const KvCost apart = kv_cost(heads, rows, 1, pre_kt);
    x.one = g_use_wide.load(std::memory_order_relaxed) != 2 && here - std::min(apart.narrow, apart.wide) < 7.0;
  }
  if (prefix > 0 && (x.one || x.own.nt == 0)) {
    const KvPass both = kv_pass(heads, rows, seqs, own_kt + pre_kt, KV_PLAIN_COST);
    x.one = x.own.nt == 0 || both.nt;   // many rows are worked on with the prefix's tiles, if at all
    if (x.one) x.own = both;
  }
  x.part = take(x.own.grid * 2 * (x.own.nt ? x.own.bm * D + 2 * x.own.bm : kv_wide_part_floats(D)) * sizeof(float));
  if (prefix > 0 && !x.one) {
    x.pre = kv_pass(heads, rows, 1, pre_kt, KV_PLAIN_COST);
    const int64_t units = heads * ((rows + x.pre.bm - 1) / x.pre.bm);
    x.pre_unit = x.pre.nt ? x.pre.cost + pre_kt : KV_WIDE_UNIT_COST + prefix;   // in tiles or in keys
    x.pre_first = x.pre.nt ? x.pre.cost : KV_WIDE_UNIT_COST;
    x.pre_last = x.pre.nt ? x.pre.cost + pre_kt - 1 : KV_WIDE_UNIT_COST + (pre_kt - 1) * TK;
    x.pre.w = units * x.pre_unit;
    x.pre.grid = kv_grid(units, pre_kt, x.pre.nt == 0 ? 1 : x.pre.nt == 1 ? 3 : 2);
    x.pre_run = (x.pre.w + x.pre.grid - 1) / x.pre.grid;
    if (x.pre.nt == 0 && x.pre_run < TK) x.pre_run = TK;
    x.pre_splits = (x.pre_last - x.pre_first) / x.pre_run + 2;
    if (x.pre_splits > pre_kt) x.pre_splits = pre_kt;
    x.pre_ml = take((x.pre_splits * heads * rows + 32) * 2 * sizeof(float));   // windows of m and l begin at even rows and end behind a unit's
    x.pre_o = take(x.pre_splits * heads * rows * D * sizeof(float));
  }
  return x;
}

}  // namespace
}  // namespace rh3

using namespace rh3;

extern "C" int64_t rh3_kv_attn_workspace_bytes(int64_t heads, int64_t group, int64_t page, int64_t D, int64_t per_seq, int64_t B, int64_t T,
                                               int64_t prefix) {
  if (heads <= 0 || group <= 0 || page <= 0 || (D != 64 && D != 128) || per_seq < 0 || B <= 0 || T <= 0 || prefix < 0) return 0;
  return kv_plan(heads, group, page, D, per_seq, B, T, prefix).bytes;
}

extern "C" int rh3_kv_attn_launches(int64_t heads, int64_t group, int64_t page, int64_t D, int64_t per_seq, int64_t B, int64_t T, int64_t prefix) {
  if (heads <= 0 || group <= 0 || page <= 0 || (D != 64 && D != 128) || per_seq < 0 || B <= 0 || T <= 0 || prefix < 0) return 0;
  return kv_plan(heads, group, page, D, per_seq, B, T, prefix).pre.grid ? 2 : 1;
}

extern "C" int rh3_kv_attn_use_wide(int use) { return g_use_wide.exchange(use < 0 || use > 2 ? -1 : use); }

extern "C" int rh3_kv_attn(const rh3_kv_attn_args* a, void* workspace, int64_t workspace_bytes, int32_t* counters, cudaStream_t stream) {
  RH3_CHECK_ARG(a, "kv_attn: null arguments");
  KvAttnParams p{};
  if (int e = kv_fill_cache(&p.c, "kv_attn", a->k, a->v, a->ks, a->vs, a->pages, a->heads, a->page, a->D, a->kind)) return e;
  if (int e = kv_fill_rows(&p.r, "kv_attn", a->table, a->table_stride, a->per_seq, a->lens, a->starts, a->B, a->T)) return e;
  RH3_CHECK_ARG(a->dtype == 0 || a->dtype == 1, "kv_attn: dtype=%d must be 0 (bf16) or 1 (fp16)", a->dtype);
  RH3_CHECK_ARG(a->group >= 1 && a->group <= 4096 && a->group * a->heads <= 4096, "kv_attn: %lld query heads per KV head", (long long)a->group);
  RH3_CHECK_ARG(a->scale > 0.f && a->scale < INFINITY, "kv_attn: the softmax scale must be positive and finite");
  RH3_CHECK_ARG(a->prefix >= 0 && a->prefix <= a->prefix_pages * a->page && (a->prefix == 0 || a->prefix_table),
                "kv_attn: a prefix of %lld tokens needs a table of its pages", (long long)a->prefix);
  if (a->T == 0) return 0;
  RH3_CHECK_ARG(a->T * a->group < (1ll << 31), "kv_attn: too many rows");
  RH3_CHECK_ARG(a->q && a->out && kv_a16(a->q) && kv_a16(a->out) && a->q_st % 8 == 0 && a->q_sh % 8 == 0 && a->o_st % 8 == 0 && a->o_sh % 8 == 0,
                "kv_attn: every row of q and out must start on a 16-byte boundary");
  const KvPlan x = kv_plan(a->heads, a->group, a->page, a->D, a->per_seq, a->B, a->T, a->prefix);
  RH3_CHECK_ARG(workspace && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0 && workspace_bytes >= x.bytes,
                "kv_attn: a workspace of %lld bytes, 256-byte aligned, is needed", (long long)x.bytes);
  RH3_CHECK_ARG(counters && x.own.grid <= RH3_KV_COUNTERS, "kv_attn: the counters are missing, or too few for the device");
  RH3_CHECK_ARG(x.own.w < (1ll << 31) && x.pre.w < (1ll << 31), "kv_attn: too many rows x tokens for one call");
  p.q = static_cast<const uint16_t*>(a->q);
  p.out = static_cast<uint16_t*>(a->out);
  p.q_st = a->q_st, p.q_sh = a->q_sh, p.o_st = a->o_st, p.o_sh = a->o_sh;
  p.is_f16 = a->dtype;
  p.group = static_cast<int>(a->group);
  p.causal = a->causal != 0;
  p.sl2 = static_cast<float>(static_cast<double>(a->scale) * 1.4426950408889634);
  p.status = device_status_word();
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.count = counters;
  p.cost = x.own.cost;
  p.part = reinterpret_cast<float*>(ws + x.part);
  if (x.one) {
    p.r.pre_tiles = static_cast<int>((a->prefix + TK - 1) / TK);
    p.pre_table = a->prefix_table;
    p.pre_len = static_cast<int>(a->prefix);
  }
  if (x.own.nt == 0) return kv_wide_launch(p, a->D, a->kind, false, x.own.grid, stream);
  CUtensorMap mk, mv;
  if (int e = kv_maps(&mk, &mv, p.c, a->D)) return e;
  auto launch = [&](auto mode, const KvAttnParams& q, const KvPass& pass) {
    constexpr int M = decltype(mode)::value;
    auto by_kind = [&](auto d, auto n) {
      constexpr int DD = decltype(d)::value, N = decltype(n)::value;
      return a->kind == RH3_KIND_I8 ? kv_launch<DD, RH3_KIND_I8, M, N>(mk, mv, q, pass.grid, stream) : kv_launch<DD, RH3_KIND_F8, M, N>(mk, mv, q, pass.grid, stream);
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    if (a->D == 128) return pass.nt == 1 ? by_kind(std::integral_constant<int, 128>(), One()) : by_kind(std::integral_constant<int, 128>(), Two());
    return pass.nt == 1 ? by_kind(std::integral_constant<int, 64>(), One()) : by_kind(std::integral_constant<int, 64>(), Two());
  };
  if (a->prefix == 0) return launch(std::integral_constant<int, MODE_PLAIN>(), p, x.own);
  if (x.one) return launch(std::integral_constant<int, MODE_ONE>(), p, x.own);
  p.pre_ml = reinterpret_cast<float*>(ws + x.pre_ml);
  p.pre_o = reinterpret_cast<float*>(ws + x.pre_o);
  p.pre_unit = static_cast<int>(x.pre_unit);
  p.pre_first = static_cast<int>(x.pre_first);
  p.pre_last = static_cast<int>(x.pre_last);
  p.pre_bm = static_cast<int>(x.pre.bm);
  p.pre_run = static_cast<int>(x.pre_run);
  // the prefix is one sequence whose rows are all rows of the call
  KvAttnParams q = p;
  q.r = KvRows{a->prefix_table, nullptr, nullptr, a->prefix_pages, 1, static_cast<int>(a->prefix_pages), static_cast<int>(a->T),
               static_cast<int>(a->prefix), 0};
  q.causal = 0;
  q.cost = x.pre.cost;
  if (int e = x.pre.nt == 0 ? kv_wide_launch(q, a->D, a->kind, true, x.pre.grid, stream) : launch(std::integral_constant<int, MODE_PREFIX>(), q, x.pre)) return e;
  return launch(std::integral_constant<int, MODE_OWN>(), p, x.own);
}
