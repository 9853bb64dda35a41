// Attention of few rows per sequence (decoding, short continuations) to the quantized paged cache.
//
// A unit is 16 rows (new tokens x query heads of one KV head) of one sequence against all of its keys. What bounds it is reading the
// cache once: 2 * (D + 4) bytes per key and head. The key tiles of all units are dealt to the CTAs in equal runs (kv_cache.cuh), two CTAs per
// SM, so ragged batches, single sequences and many heads all spread over the chip; a unit cut by a run's end leaves partial results
// that a second small kernel joins in a fixed order.
//
// One CTA = a producer warp and four warps that compute, each on 32 of a tile's 128 keys with its own running maximum, sums and
// output, joined at the unit's end: no barrier among them per tile. The producer brings pages by TMA into a ring
// (128-byte swizzle over the codes as they lie, so that the byte accesses below hit 32 banks), their scales by bulk copies.
// Products are mma.sync m16n8k16 on fp16: 16 rows are all there is, a 128-row tensor-core tile would be seven-eighths empty,
// and the conversion of the codes (5 instructions per 4 codes) costs more than the products.
// The order of channels and keys inside an mma is free, so each lane takes the channels and keys whose bytes it can load
// 16 at a time: channel order (K) 16c .. 16c+15 of lane c, key order n -> (n >> 1) | ((n & 1) << 2), output channels of
// lane group g 16g' .. 16g'+15.
#include "kv_attn.cuh"
#include "rapidh3_b200.h"

namespace rh3 {
namespace {

constexpr int TK = 128;                 // keys of a tile
constexpr int KV_WARPS = 4;             // computing warps
constexpr int KV_NT = KV_WARPS * 32 + 32;
enum { MODE_PLAIN = 0, MODE_PREFIX = 1, MODE_OWN = 2 };

template <int D>
struct KvNarrow {
  static constexpr int STAGES = D == 128 ? 3 : 5;
  static constexpr int STAGE_BYTES = 2 * TK * D;
  static constexpr int SCALES = STAGES * STAGE_BYTES;             // [STAGES][2][TK] floats
  static constexpr int MERGE = SCALES + STAGES * 2 * TK * 4;      // [D / 8][32] float4
  static constexpr int TAIL = MERGE + KV_BM * D * 4;
};
struct __align__(8) KvTail {
  uint64_t full[5], empty[5];
  float ml[KV_WARPS][KV_BM][2];
  long long scan[KV_NT / 32];
  KvRun run;
  uint32_t pages[5];   // which of a stage's pages were there
  int abort_flag;
};
template <int D>
constexpr int kv_narrow_smem() { return KvNarrow<D>::TAIL + static_cast<int>(sizeof(KvTail)) + 1024; }

__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// after an abandoned wait: copies that are still on their way land before the CTA gives its shared memory back
__device__ __forceinline__ void kv_settle() {
  for (int i = 0; i < 64; ++i) __nanosleep(1000);
}

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
  long long flat; // row number in the prefix pass
};
__device__ __forceinline__ KvLaneRow kv_lane_row(const KvAttnParams& p, const KvSegment& g, int r) {
  KvLaneRow x;
  const long long flat = static_cast<long long>(g.u) * KV_BM + r;
  const int i = static_cast<int>(flat / p.group), hh = static_cast<int>(flat - static_cast<long long>(i) * p.group);
  const bool there = i < g.s.n;
  const int64_t t = g.s.first + i, head = static_cast<int64_t>(g.h) * p.group + hh;
  x.q = there ? t * p.q_st + head * p.q_sh : -1;
  x.o = t * p.o_st + head * p.o_sh;
  x.pos = p.causal ? g.s.len - g.s.n + i : g.s.len - 1;
  x.flat = t * p.group + hh;
  return x;
}
__device__ __forceinline__ float2 kv_unpack(uint32_t w, int is_f16) {
  if (is_f16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(bf16_lo(w), bf16_hi(w));
}
__device__ __forceinline__ uint32_t kv_pack(float a, float b, int is_f16) { return is_f16 ? pack_half2(a, b) : pack_bf16x2(a, b); }

template <int D, int FMT, int MODE>
__global__ void __launch_bounds__(KV_NT, 2)
kv_attn_kernel(const __grid_constant__ CUtensorMap tma_k, const __grid_constant__ CUtensorMap tma_v, const KvAttnParams p) {
  using L = KvNarrow<D>;
  constexpr int S = L::STAGES, NJ = D / 8, CH = D / 8, QW = D / 4;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* scales = reinterpret_cast<float*>(smem + L::SCALES);
  float4* merge = reinterpret_cast<float4*>(smem + L::MERGE);
  KvTail* tail = reinterpret_cast<KvTail*>(smem + L::TAIL);
  volatile int* abort_flag = &tail->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&tail->full[s], 1);
      mbar_init(&tail->empty[s], KV_WARPS);
    }
    tail->abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  grid_dependency_begin();
  kv_find_run<KV_BM, TK, KV_NT>(p.r, p.c.page_log2, p.c.heads, p.group, tail->scan, &tail->run);
  KvWalk<KV_BM, TK> walk(tail->run);
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
    while (walk.next(p.r, p.c.page_log2, p.c.heads, p.group, g)) {
      const int kend = min(g.k1, (kv_visible<KV_BM>(g.s, p.group, g.u, p.causal) + TK - 1) / TK);
      for (int kt = g.k0; kt < kend; ++kt) {
        const int at = kt * tile_pages + lane;
        const bool need = lane < tile_pages && (static_cast<int64_t>(at) << p.c.page_log2) < g.s.len;
        const int id = need ? p.r.table[g.b * p.r.table_stride + at] : -1;
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
  const int gq = lane >> 2, c = lane & 3;   // row pair gq, gq + 8; quarter of the channels / keys
  const int kc0 = col_perm<D>(2 * c), kc1 = col_perm<D>(2 * c + 1);
  bool ok = true, first = true;
  int stage = 0;
  uint32_t ph = 0;
  if (MODE != MODE_PREFIX && threadIdx.x == 0 && tail->run.x0 >= tail->run.x1) p.record[2 * blockIdx.x] = make_int4(-1, 0, 0, 0);
  while (walk.next(p.r, p.c.page_log2, p.c.heads, p.group, g)) {
    if (MODE != MODE_PREFIX && first && threadIdx.x == 0) {
      p.record[2 * blockIdx.x] = make_int4(g.k0 > 0 ? g.b : -1, g.h, g.u, g.s.kt);
      const unsigned long long W = static_cast<unsigned long long>(tail->run.W);
      p.record[2 * blockIdx.x + 1] = make_int4(g.k0, static_cast<int>(W & 0xffffffffu), static_cast<int>(W >> 32), tail->run.G);
    }
    first = false;
    const KvLaneRow r0 = kv_lane_row(p, g, gq), r1 = kv_lane_row(p, g, gq + 8);
    // q rows: channels 16c .. 16c+15 of each 64, as the A fragments of D / 16 products
    uint32_t a[D / 16][4];
    float c0, c1;
    {
      uint32_t x[2][QW / 2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t at = i ? r1.q : r0.q;
#pragma unroll
        for (int j = 0; j < QW / 8; ++j) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (at >= 0) v = ld_global_16(p.q + at + (j >> 1) * 64 + c * 16 + (j & 1) * 8);
          x[i][4 * j] = v.x, x[i][4 * j + 1] = v.y, x[i][4 * j + 2] = v.z, x[i][4 * j + 3] = v.w;
        }
      }
      float up[2], down[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < QW / 2; ++j) {
          const float2 f = kv_unpack(x[i][j], p.is_f16);
          amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        kv_row_factor(amax, up[i], down[i]);
#pragma unroll
        for (int j = 0; j < QW / 2; ++j) {
          const float2 f = kv_unpack(x[i][j], p.is_f16);
          a[j >> 1][i + 2 * (j & 1)] = pack_half2(f.x * up[i], f.y * up[i]);
        }
      }
      c0 = p.sl2 * down[0], c1 = p.sl2 * down[1];
    }
    float o[NJ][4];
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    const int kend = min(g.k1, (kv_visible<KV_BM>(g.s, p.group, g.u, p.causal) + TK - 1) / TK);
    const int pos_first = p.causal ? g.s.len - g.s.n + static_cast<int>(static_cast<long long>(g.u) * KV_BM / p.group) : g.s.len - 1;
    for (int kt = g.k0; kt < kend; ++kt) {
      if (!__all_sync(0xffffffffu, mbar_wait(&tail->full[stage], ph, abort_flag, p.status, ST_TIMEOUT_TMA_FULL))) {
        ok = false;
        break;
      }
      uint8_t* sk = smem + stage * L::STAGE_BYTES + warp * 32 * D;
      uint8_t* sv = sk + TK * D;
      const float* sks = scales + stage * 2 * TK + warp * 32;
      const uint32_t pages = tail->pages[stage];
      const int key0 = warp * 32, pos0 = kt * TK + key0;
      const bool whole = pages == (0xffffffffu >> (32 - (TK >> p.c.page_log2))) && kt * TK + TK <= g.s.len;
      const bool masked = !whole || kt * TK + TK - 1 > pos_first;
      auto there = [&](int key) { return pos0 + key < g.s.len && ((pages >> ((key0 + key) >> p.c.page_log2)) & 1u); };
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
      // ---- scores: 4 blocks of 8 keys ----
      float u[4][4];
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) {
        const int key = nb * 8 + col_perm<D>(gq);
        uint32_t w[QW / 4];
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const uint4 v = *reinterpret_cast<const uint4*>(sk + chunk_at<D>(key, 4 * i + c));
          w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
        u[nb][0] = u[nb][1] = u[nb][2] = u[nb][3] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          uint32_t b0, b1;
          kv_codes_to_half<FMT>(w[j], b0, b1);
          mma_f16(u[nb], a[j], b0, b1);
        }
      }
      float iv[4][2];
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = nb * 8 + (e ? kc1 : kc0);
          const float ks = sks[key], vs = fmaxf(sks[TK + key], kVsMin);
          const float lv = kv_lg2(vs);
          iv[nb][e] = __frcp_rn(vs);
          u[nb][e] = fmaf(u[nb][e] * ks, c0, lv);
          u[nb][2 + e] = fmaf(u[nb][2 + e] * ks, c1, lv);
          if (masked) {
            const bool is = there(key);
            if (!is || pos0 + key > r0.pos) u[nb][e] = -INFINITY;
            if (!is || pos0 + key > r1.pos) u[nb][2 + e] = -INFINITY;
          }
        }
      }
      // ---- running maximum ----
      float n0 = m0, n1 = m1;
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) {
        n0 = fmaxf(n0, fmaxf(u[nb][0], u[nb][1]));
        n1 = fmaxf(n1, fmaxf(u[nb][2], u[nb][3]));
      }
      n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 1));
      n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 1));
      n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 2));
      n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 2));
      const float z0 = n0 == -INFINITY ? 0.f : n0, z1 = n1 == -INFINITY ? 0.f : n1;   // nothing seen yet: weights 2^-inf = 0
      if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {
        const float f0 = kv_ex2(m0 - z0), f1 = kv_ex2(m1 - z1);
        l0 *= f0, l1 *= f1;
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[j][0] *= f0, o[j][1] *= f0, o[j][2] *= f1, o[j][3] *= f1;
        m0 = n0, m1 = n1;
      }
      // ---- weights ----
      uint32_t pa[2][4];
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = kv_ex2(u[nb][e] - (e < 2 ? z0 : z1) + kWeightLog2);
          // a masked key's 1 / vs may be anything
          const float add = masked && w[e] == 0.f ? 0.f : w[e] * iv[nb][e & 1];
          if (e < 2) l0 += add;
          else l1 += add;
        }
        pa[nb >> 1][2 * (nb & 1)] = pack_half2(w[0], w[1]);
        pa[nb >> 1][2 * (nb & 1) + 1] = pack_half2(w[2], w[3]);
      }
      // ---- O += w . V: 2 steps of 16 keys ----
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        constexpr int VW = D / 32;   // words of D / 8 channels
        uint32_t v[4][VW];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = s * 16 + (i >> 1) * 8 + ((i & 1) ? kc1 : kc0);
          if constexpr (D == 128) {
            const uint4 x = *reinterpret_cast<const uint4*>(sv + chunk_at<D>(key, col_perm<D>(gq)));
            v[i][0] = x.x, v[i][1] = x.y, v[i][2] = x.z, v[i][3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(sv + chunk_at<D>(key, gq >> 1) + (gq & 1) * 8);
            v[i][0] = x.x, v[i][1] = x.y;
          }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          uint32_t b0[4], b1[4];
          kv_codes_to_half<FMT>(__byte_perm(v[0][w], v[1][w], 0x5140), b0[0], b0[1]);
          kv_codes_to_half<FMT>(__byte_perm(v[0][w], v[1][w], 0x7362), b0[2], b0[3]);
          kv_codes_to_half<FMT>(__byte_perm(v[2][w], v[3][w], 0x5140), b1[0], b1[1]);
          kv_codes_to_half<FMT>(__byte_perm(v[2][w], v[3][w], 0x7362), b1[2], b1[3]);
#pragma unroll
          for (int b = 0; b < 4; ++b) mma_f16(o[4 * w + b], pa[s], b0[b], b1[b]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&tail->empty[stage]);
      if (++stage == S) stage = 0, ph ^= 1;
    }

    // what the prefix pass found for these rows joins in the part that begins the unit; warp w takes splits w, w + 4, ...
    if (MODE == MODE_OWN && g.k0 == 0) {
      const long long rows = static_cast<long long>(p.r.T) * p.group;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const KvLaneRow& r = i ? r1 : r0;
        float& m = i ? m1 : m0;
        float& l = i ? l1 : l0;
        int n = 0;
        if (r.q >= 0) {
          const long long unit = static_cast<long long>(g.h) * ((rows + p.pre_bm - 1) / p.pre_bm) + r.flat / p.pre_bm;
          n = kv_owner(unit * p.pre_kt + p.pre_kt - 1, p.pre_w, p.pre_g) - kv_owner(unit * p.pre_kt, p.pre_w, p.pre_g) + 1;
        }
        for (int s = warp; s < n; s += KV_WARPS) {
          const long long at = (static_cast<long long>(s) * p.c.heads + g.h) * rows + r.flat;
          const float pm = p.pre_ml[2 * at], pl = p.pre_ml[2 * at + 1];
          const float nm = fmaxf(m, pm);
          const float z = nm == -INFINITY ? 0.f : nm;
          const float f = kv_ex2(m - z), fp = kv_ex2(pm - z);
          m = nm;
          l = l * f + (c == 0 ? pl * fp : 0.f);   // l is a sum over the row's four lanes
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float* src = p.pre_o + at * D + CH * (e ? kc1 : kc0);
#pragma unroll
            for (int j = 0; j < CH; j += 4) {
              const uint4 x = ld_global_16(src + j);
              o[j][2 * i + e] = o[j][2 * i + e] * f + __uint_as_float(x.x) * fp;
              o[j + 1][2 * i + e] = o[j + 1][2 * i + e] * f + __uint_as_float(x.y) * fp;
              o[j + 2][2 * i + e] = o[j + 2][2 * i + e] * f + __uint_as_float(x.z) * fp;
              o[j + 3][2 * i + e] = o[j + 3][2 * i + e] * f + __uint_as_float(x.w) * fp;
            }
          }
        }
      }
    }

    // ---- join the four warps ----
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    if (c == 0) {
      tail->ml[warp][gq][0] = m0, tail->ml[warp][gq][1] = l0;
      tail->ml[warp][gq + 8][0] = m1, tail->ml[warp][gq + 8][1] = l1;
    }
    if (bar_sync_or(1, KV_WARPS * 32, !ok)) {
      kv_settle();
      return;
    }
    float M0 = -INFINITY, M1 = -INFINITY, L0 = 0.f, L1 = 0.f;
#pragma unroll
    for (int w = 0; w < KV_WARPS; ++w) M0 = fmaxf(M0, tail->ml[w][gq][0]), M1 = fmaxf(M1, tail->ml[w][gq + 8][0]);
    const float z0 = M0 == -INFINITY ? 0.f : M0, z1 = M1 == -INFINITY ? 0.f : M1;
#pragma unroll
    for (int w = 0; w < KV_WARPS; ++w) {
      L0 += tail->ml[w][gq][1] * kv_ex2(tail->ml[w][gq][0] - z0);
      L1 += tail->ml[w][gq + 8][1] * kv_ex2(tail->ml[w][gq + 8][0] - z1);
    }
    const float f0 = kv_ex2(m0 - z0), f1 = kv_ex2(m1 - z1);
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j][0] *= f0, o[j][1] *= f0, o[j][2] *= f1, o[j][3] *= f1;
#pragma unroll
    for (int w = 1; w <= KV_WARPS; ++w) {   // warp 1 writes, 2 and 3 add in place, 0 takes the sum
      if (warp == (w & (KV_WARPS - 1))) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          if (w > 1) {
            const float4 x = merge[j * 32 + lane];
            o[j][0] += x.x, o[j][1] += x.y, o[j][2] += x.z, o[j][3] += x.w;
          }
          if (w < KV_WARPS) merge[j * 32 + lane] = make_float4(o[j][0], o[j][1], o[j][2], o[j][3]);
        }
      }
      if (w < KV_WARPS) asm volatile("bar.sync 2, %0;" ::"n"(KV_WARPS * 32) : "memory");
    }
    if (warp != 0) continue;

    if constexpr (MODE == MODE_PREFIX) {
      const long long rows = static_cast<long long>(p.r.T) * p.group;
      const long long unit = static_cast<long long>(g.h) * g.s.qt + g.u;
      const int s = blockIdx.x - kv_owner(unit * g.s.kt, tail->run.W, tail->run.G);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const KvLaneRow& r = i ? r1 : r0;
        if (r.q < 0) continue;
        const long long at = (static_cast<long long>(s) * p.c.heads + g.h) * rows + r.flat;
        if (c == 0) p.pre_ml[2 * at] = i ? M1 : M0, p.pre_ml[2 * at + 1] = i ? L1 : L0;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float4* dst = reinterpret_cast<float4*>(p.pre_o + at * D + CH * (e ? kc1 : kc0));
#pragma unroll
          for (int j = 0; j < CH; j += 4)
            dst[j >> 2] = make_float4(o[j][2 * i + e], o[j + 1][2 * i + e], o[j + 2][2 * i + e], o[j + 3][2 * i + e]);
        }
      }
    } else if (g.k0 == 0 && g.k1 == g.s.kt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const KvLaneRow& r = i ? r1 : r0;
        if (r.q < 0) continue;
        const float l = i ? L1 : L0;
        const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);   // no key: 0
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint16_t* dst = p.out + r.o + CH * (e ? kc1 : kc0);
#pragma unroll
          for (int j = 0; j < CH; j += 8) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = kv_pack(o[j + 2 * k][2 * i + e] * inv, o[j + 2 * k + 1][2 * i + e] * inv, p.is_f16);
            *reinterpret_cast<uint4*>(dst + j) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    } else {
      float* slot = p.part + (2ll * blockIdx.x + (g.k0 > 0 ? 0 : 1)) * kv_part_floats<D>();
#pragma unroll
      for (int j = 0; j < NJ; ++j) reinterpret_cast<float4*>(slot)[j * 32 + lane] = make_float4(o[j][0], o[j][1], o[j][2], o[j][3]);
      if (c == 0) {
        float* ml = slot + KV_BM * D;
        ml[gq] = M0, ml[gq + 8] = M1;
        ml[KV_BM + gq] = L0, ml[KV_BM + gq + 8] = L1;
      }
    }
  }
}

// Joins the parts of the unit that CTA c = blockIdx.x + 1 of the pass before began inside of, if it was the first to do so:
// slot 1 of CTA c - 1 and slot 0 of c, c + 1, ... while their runs begin inside the unit. Parts are taken in order.
template <int D>
__global__ void __launch_bounds__(4 * D) kv_join_kernel(const KvAttnParams p) {
  __shared__ float rows[KV_BM][D + 4];
  grid_dependency_begin();
  const int c = blockIdx.x + 1;
  const int4 a = p.record[2 * c];
  if (a.x < 0) return;
  const int4 r = p.record[2 * c + 1];
  const long long W = static_cast<long long>((static_cast<unsigned long long>(static_cast<unsigned>(r.z)) << 32) | static_cast<unsigned>(r.y));
  const int G = r.w;
  const long long xs = W * c / G - r.x, xe = xs + a.w;
  if (W * (c - 1) / G > xs) return;
  const int n = kv_owner(xe - 1, W, G) - c + 2;
  const int lane = threadIdx.x & 31, j = threadIdx.x >> 5, gq = lane >> 2, q = lane & 3;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int STEP = 8;
  for (int i0 = 0; i0 < n; i0 += STEP) {
    float4 x[STEP];
    float pm[STEP][2], pl[STEP][2];
#pragma unroll
    for (int i = 0; i < STEP; ++i) {
      if (i0 + i < n) {
        const float* slot = p.part + (i0 + i == 0 ? 2ll * (c - 1) + 1 : 2ll * (c - 1 + i0 + i)) * kv_part_floats<D>();
        x[i] = reinterpret_cast<const float4*>(slot)[j * 32 + lane];
        pm[i][0] = slot[KV_BM * D + gq], pm[i][1] = slot[KV_BM * D + gq + 8];
        pl[i][0] = slot[KV_BM * D + KV_BM + gq], pl[i][1] = slot[KV_BM * D + KV_BM + gq + 8];
      } else {
        x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        pm[i][0] = pm[i][1] = -INFINITY, pl[i][0] = pl[i][1] = 0.f;
      }
    }
    float n0 = m0, n1 = m1;
#pragma unroll
    for (int i = 0; i < STEP; ++i) n0 = fmaxf(n0, pm[i][0]), n1 = fmaxf(n1, pm[i][1]);
    const float z0 = n0 == -INFINITY ? 0.f : n0, z1 = n1 == -INFINITY ? 0.f : n1;
    const float f0 = kv_ex2(m0 - z0), f1 = kv_ex2(m1 - z1);
    o.x *= f0, o.y *= f0, o.z *= f1, o.w *= f1, l0 *= f0, l1 *= f1;
    m0 = n0, m1 = n1;
#pragma unroll
    for (int i = 0; i < STEP; ++i) {
      const float e0 = kv_ex2(pm[i][0] - z0), e1 = kv_ex2(pm[i][1] - z1);
      o.x += x[i].x * e0, o.y += x[i].y * e0, o.z += x[i].z * e1, o.w += x[i].w * e1;
      l0 += pl[i][0] * e0, l1 += pl[i][1] * e1;
    }
  }
  const float i0 = l0 == 0.f ? 0.f : __fdiv_rn(1.f, l0), i1 = l1 == 0.f ? 0.f : __fdiv_rn(1.f, l1);
  constexpr int CH = D / 8;
  rows[gq][CH * col_perm<D>(2 * q) + j] = o.x * i0;
  rows[gq][CH * col_perm<D>(2 * q + 1) + j] = o.y * i0;
  rows[gq + 8][CH * col_perm<D>(2 * q) + j] = o.z * i1;
  rows[gq + 8][CH * col_perm<D>(2 * q + 1) + j] = o.w * i1;
  __syncthreads();
  KvSegment g;
  g.s = kv_seq<KV_BM, TK>(p.r, p.c.page_log2, p.group, a.x);
  g.b = a.x, g.h = a.y, g.u = a.z;
  for (int k = threadIdx.x; k < KV_BM * D / 8; k += 4 * D) {
    const int row = k / (D / 8), ch = (k % (D / 8)) * 8;
    const KvLaneRow x = kv_lane_row(p, g, row);
    if (x.q < 0) continue;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = kv_pack(rows[row][ch + 2 * i], rows[row][ch + 2 * i + 1], p.is_f16);
    *reinterpret_cast<uint4*>(p.out + x.o + ch) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

int kv_maps(CUtensorMap* mk, CUtensorMap* mv, const KvCache& c, int64_t D) {
  const uint64_t page = 1ull << c.page_log2, rows = static_cast<uint64_t>(c.pages) * c.heads * page * D / 128;
  const uint32_t box = static_cast<uint32_t>(page * D / 128);
  if (int e = make_tmap_2d(mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.k, 128, rows, 128, 128, box, CU_TENSOR_MAP_SWIZZLE_128B)) return e;
  return make_tmap_2d(mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.v, 128, rows, 128, 128, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// CTAs of a pass: two per SM, no more than there can be tiles
template <class I>
I kv_grid(I units, I kt) {
  const I most = 2 * static_cast<I>(device_sm_count());
  return units * kt < most ? units * kt : most;
}

template <int D, int FMT, int MODE>
int kv_launch(const CUtensorMap& mk, const CUtensorMap& mv, const KvAttnParams& p, int64_t grid, cudaStream_t stream) {
  auto kern = kv_attn_kernel<D, FMT, MODE>;
  const int smem = kv_narrow_smem<D>();
  if (int e = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "kv_attn smem attribute")) return e;
  return check_cuda(launch_chained(kern, dim3(static_cast<unsigned>(grid)), KV_NT, smem, stream, 1, mk, mv, p), "kv_attn launch");
}

// The plan of a call: grids and the pieces of its workspace
struct KvPlan {
  int64_t kt, grid, pre_kt, pre_grid, pre_splits;   // own pass; prefix pass
  int64_t record, part, pre_ml, pre_o, bytes;       // byte offsets
};
KvPlan kv_plan(int64_t heads, int64_t group, int64_t page, int64_t D, int64_t per_seq, int64_t B, int64_t T, int64_t prefix) {
  KvPlan x{};
  const int64_t rows = T * group;
  x.kt = (per_seq * page + TK - 1) / TK;
  if (x.kt < 1) x.kt = 1;
  x.grid = kv_grid<int64_t>(heads * (rows / KV_BM + (B < T ? B : T)), x.kt);
  auto take = [&](int64_t bytes) {
    const int64_t at = x.bytes;
    x.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  x.record = take(x.grid * 2 * sizeof(int4));
  x.part = take(x.grid * 2 * (D == 128 ? kv_part_floats<128>() : kv_part_floats<64>()) * sizeof(float));
  if (prefix > 0) {
    const int64_t units = heads * ((rows + KV_BM - 1) / KV_BM);
    x.pre_kt = (prefix + TK - 1) / TK;
    x.pre_grid = kv_grid<int64_t>(units, x.pre_kt);
    const int64_t run = units * x.pre_kt / x.pre_grid;    // tiles of the shortest run
    x.pre_splits = (x.pre_kt - 1) / run + 2;
    if (x.pre_splits > x.pre_kt) x.pre_splits = x.pre_kt;
    x.pre_ml = take(x.pre_splits * heads * rows * 2 * sizeof(float));
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

extern "C" int rh3_kv_attn(const rh3_kv_attn_args* a, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  RH3_CHECK_ARG(a, "kv_attn: null arguments");
  KvAttnParams p{};
  if (int e = kv_fill_cache(&p.c, "kv_attn", a->k, a->v, a->ks, a->vs, a->pages, a->heads, a->page, a->D, a->kind)) return e;
  if (int e = kv_fill_rows(&p.r, "kv_attn", a->table, a->table_stride, a->per_seq, a->lens, a->starts, a->B, a->T)) return e;
  RH3_CHECK_ARG(a->dtype == 0 || a->dtype == 1, "kv_attn: dtype=%d must be 0 (bf16) or 1 (fp16)", a->dtype);
  RH3_CHECK_ARG(a->group >= 1 && a->group * a->heads <= 4096, "kv_attn: %lld query heads per KV head", (long long)a->group);
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
  p.q = static_cast<const uint16_t*>(a->q);
  p.out = static_cast<uint16_t*>(a->out);
  p.q_st = a->q_st, p.q_sh = a->q_sh, p.o_st = a->o_st, p.o_sh = a->o_sh;
  p.is_f16 = a->dtype;
  p.group = static_cast<int>(a->group);
  p.causal = a->causal != 0;
  p.sl2 = static_cast<float>(static_cast<double>(a->scale) * 1.4426950408889634);
  p.status = device_status_word();
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.record = reinterpret_cast<int4*>(ws + x.record);
  p.part = reinterpret_cast<float*>(ws + x.part);
  CUtensorMap mk, mv;
  if (int e = kv_maps(&mk, &mv, p.c, a->D)) return e;

  auto launch = [&](auto mode, const KvAttnParams& q, int64_t grid) {
    constexpr int M = decltype(mode)::value;
    if (a->D == 128)
      return a->kind == RH3_KIND_I8 ? kv_launch<128, RH3_KIND_I8, M>(mk, mv, q, grid, stream) : kv_launch<128, RH3_KIND_F8, M>(mk, mv, q, grid, stream);
    return a->kind == RH3_KIND_I8 ? kv_launch<64, RH3_KIND_I8, M>(mk, mv, q, grid, stream) : kv_launch<64, RH3_KIND_F8, M>(mk, mv, q, grid, stream);
  };
  if (a->prefix > 0) {
    p.pre_ml = reinterpret_cast<float*>(ws + x.pre_ml);
    p.pre_o = reinterpret_cast<float*>(ws + x.pre_o);
    p.pre_kt = static_cast<int>(x.pre_kt);
    p.pre_bm = KV_BM;
    p.pre_w = a->heads * ((a->T * a->group + KV_BM - 1) / KV_BM) * x.pre_kt;
    p.pre_g = static_cast<int>(x.pre_grid);
    // the prefix is one sequence whose rows are all rows of the call
    KvAttnParams q = p;
    q.r = KvRows{a->prefix_table, nullptr, nullptr, a->prefix_pages, 1, static_cast<int>(a->prefix_pages), static_cast<int>(a->T),
                 static_cast<int>(a->prefix)};
    q.causal = 0;
    if (int e = launch(std::integral_constant<int, MODE_PREFIX>(), q, x.pre_grid)) return e;
    if (int e = launch(std::integral_constant<int, MODE_OWN>(), p, x.grid)) return e;
  } else if (int e = launch(std::integral_constant<int, MODE_PLAIN>(), p, x.grid)) {
    return e;
  }
  if (x.kt == 1 || x.grid == 1) return 0;   // no unit can be cut
  const unsigned blocks = static_cast<unsigned>(x.grid - 1);
  return check_cuda(a->D == 128 ? launch_chained(kv_join_kernel<128>, dim3(blocks), 512, 0, stream, 1, p)
                                : launch_chained(kv_join_kernel<64>, dim3(blocks), 256, 0, stream, 1, p),
                    "kv_join launch");
}
