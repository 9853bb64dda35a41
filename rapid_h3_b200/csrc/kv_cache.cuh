// What the kernels of the quantized key/value cache share: the cache and batch descriptors, where a row of a call lies in
// the cache, and how the work of a ragged batch is cut into equal pieces on the device.
//
// Cache: codes [pages][heads][page][D] (int8 or e4m3, one byte each), scales fp32 [pages][heads][page]; page is a power of
// two of 16 .. 128 tokens, so a head's part of a page is one contiguous run that a single TMA box takes.
// Batch: table int32 [B][table_stride] (the pages of each sequence in order), lens int32 [B] (cached tokens, the call's own
// among them), starts int32 [B + 1]: rows starts[b] .. starts[b + 1] - 1 of the call are the last tokens of sequence b.
// All three live on the device and are read there: a captured call follows them when it is replayed. Values that make no
// sense (a page that does not exist, a length beyond the table, rows beyond the call's) are cut to what exists, never
// followed; a missing page's tokens count as masked, and ST_KV_BAD_PAGE is left in the status word.
#pragma once
#include "common.cuh"

namespace rh3 {

struct KvCache {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int pages, heads, page_log2;
};
struct KvRows {
  const int* table;
  const int* lens;
  const int* starts;
  int64_t table_stride;
  int B, per_seq;  // sequences; pages per row of the table
  int T;           // rows of the call
  int fixed_len;   // > 0: one sequence of this many tokens whose rows are all of the call's (a shared prefix; lens and starts are not read)
  int pre_tiles;   // key tiles of a shared prefix before every unit's own
};

// keeps a NaN, which fmaxf drops
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ void kv_report(int* status, int code) {
  if (status) atomicCAS(status, 0, code);
}

// How many of ends[0 .. n) (ascending) are <= t: a 32-way search by a whole warp, one load per lane and round (one round
// up to 32 sequences, two up to 1,024).
__device__ __forceinline__ int kv_count_ends(const int* ends, int n, int t, int lane) {
  int lo = 0;
  while (n > 0) {
    const int step = (n + 31) >> 5;
    const int first = lane * step;
    const bool have = first < n;
    const int at = lo + min(n, first + step) - 1;
    const bool below = have && ends[at] <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, below));   // chunks that lie wholly at or below t
    const int skip = min(n, c * step);
    const int left = min(step, n - skip);
    lo += skip;
    n = left > 0 ? left - 1 : 0;                               // the chunk's last element is known to be above t
  }
  return lo;
}

// Where row t of the call lies (whole warp, t uniform): pages of the cache are checked against its size.
__device__ __forceinline__ int64_t kv_place(const KvCache& c, const KvRows& r, int t, int lane, int* status, bool* known) {
  const int b = kv_count_ends(r.starts + 1, r.B, t, lane);
  *known = b < r.B && t >= r.starts[b];
  if (!*known) return -1;
  const int64_t pos = static_cast<int64_t>(r.lens[b]) - (static_cast<int64_t>(r.starts[b + 1]) - t);
  const int64_t pi = pos >> c.page_log2;
  if (pos < 0 || pi >= r.per_seq) return -1;
  const int id = r.table[b * r.table_stride + pi];
  if (id < 0 || id >= c.pages) {
    if (lane == 0) kv_report(status, ST_KV_BAD_PAGE);
    return -1;
  }
  return ((static_cast<int64_t>(id) * c.heads) << c.page_log2) + (pos & ((1 << c.page_log2) - 1));
}

// ---------------------------------------------------------------------------------------------
// cutting a ragged batch into equal pieces
// ---------------------------------------------------------------------------------------------
// The rows of a sequence are its new tokens x the query heads of one KV head ("group"): row = token * group + head. A unit is
// BM such rows of one sequence and KV head against all of its keys, in tiles of TK keys; every unit has at least one tile, so that rows
// without a key are written too. A unit weighs its tiles and `cost` more, for what it takes to begin and end it. All units, in the order
// (sequence, head, row tile), are dealt to the CTAs in runs of `run` = W / grid, rounded up: a run begins and ends anywhere inside a unit,
// where position y stands for key tile y - cost (0 up to there). W is below 2^31 (the entry refuses more) for starts that ascend;
// where they do not, sequences would claim the same rows: that is reported, and nothing is done.
struct KvSeq {
  int first, n, len;  // first row token of the call, new tokens, cached tokens
  int pos;            // position of the first row token, as kv_place has it (at most len: there it sees all of them)
  int qt, kt;         // row tiles, key tiles of a unit
  __device__ __forceinline__ unsigned weight(int heads, int cost) const { return static_cast<unsigned>(heads) * qt * (kt + cost); }
};
template <int BM, int TK>
__device__ __forceinline__ KvSeq kv_seq(const KvRows& r, int page_log2, int group, int b) {
  KvSeq s;
  const int lo = r.fixed_len ? 0 : min(max(r.starts[b], 0), r.T), end = r.fixed_len ? r.T : r.starts[b + 1], held = r.fixed_len ? r.fixed_len : r.lens[b];
  s.first = lo;
  s.n = min(max(end, lo), r.T) - lo;
  const long long room = static_cast<long long>(r.per_seq) << page_log2;
  s.len = static_cast<int>(min(static_cast<long long>(max(held, 0)), room));
  // from lens and starts as they are, not as far as the table and the call go; below 0 by more than a call has rows is all the same
  s.pos = static_cast<int>(max(-(1ll << 30), min(static_cast<long long>(s.len), held - (static_cast<long long>(end) - lo))));
  s.qt = (s.n * group + BM - 1) / BM;
  s.kt = max(1, r.pre_tiles + (s.len + TK - 1) / TK);
  return s;
}
__device__ __forceinline__ bool kv_descends(const KvRows& r, int b) { return !r.fixed_len && r.starts[b] > r.starts[b + 1]; }
struct KvRun {
  int x0, x1;   // the CTA's run
  int run;      // length of a run: x belongs to CTA x / run
  int b, xb;    // the sequence that x0 lies in and where it begins
};
// Every warp scans the sequences by itself (they are in L1 after the first): no barrier, one round of loads up to 32 sequences.
template <int BM, int TK>
__device__ __forceinline__ KvRun kv_find_run(const KvRows& r, int page_log2, int heads, int group, int cost, int* status) {
  const int lane = threadIdx.x & 31;
  const int per = (r.B + 31) >> 5;
  const int b0 = min(r.B, lane * per), b1 = min(r.B, b0 + per);
  unsigned own = 0;
  bool bad = false;
  for (int b = b0; b < b1; ++b) {
    own += kv_seq<BM, TK>(r, page_log2, group, b).weight(heads, cost);
    bad |= kv_descends(r, b);
  }
  if (__any_sync(0xffffffffu, bad)) {
    own = 0;
    if (threadIdx.x == 0) kv_report(status, ST_KV_BAD_STARTS);
  }
  unsigned total = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned up = __shfl_up_sync(0xffffffffu, total, o);
    if (lane >= o) total += up;
  }
  const int incl = static_cast<int>(total), W = __shfl_sync(0xffffffffu, incl, 31);
  KvRun run;
  run.run = max(1u, (static_cast<unsigned>(W) + gridDim.x - 1) / gridDim.x);
  run.x0 = static_cast<int>(min(static_cast<long long>(W), static_cast<long long>(run.run) * blockIdx.x));
  run.x1 = min(W - run.x0, run.run) + run.x0;
  int xb = incl - static_cast<int>(own), b = b0;
  const bool mine = run.x0 < run.x1 && xb <= run.x0 && run.x0 < incl;
  if (mine && per > 1) {
    for (; b < b1; ++b) {
      const int w = static_cast<int>(kv_seq<BM, TK>(r, page_log2, group, b).weight(heads, cost));
      if (run.x0 - xb < w) break;
      xb += w;
    }
  }
  const uint32_t who = __ballot_sync(0xffffffffu, mine);
  run.b = __shfl_sync(0xffffffffu, b, who ? __ffs(who) - 1 : 0);
  run.xb = __shfl_sync(0xffffffffu, xb, who ? __ffs(who) - 1 : 0);
  return run;
}
// One unit's part of a CTA's run
struct KvSegment {
  KvSeq s;
  int b, h, u;        // sequence, KV head, row tile
  int k0, k1;         // key tiles [k0, k1) of the unit's s.kt
  int x;              // position of the unit's first tile
};
// Steps through a run; next() gives the segment at x and moves on.
template <int BM, int TK>
struct KvWalk {
  int x, x1, xb, b;
  KvSeq s;
  bool have;
  __device__ __forceinline__ KvWalk(const KvRun& run) : x(run.x0), x1(run.x1), xb(run.xb), b(run.b), have(false) {}
  __device__ __forceinline__ bool next(const KvRows& r, int page_log2, int heads, int group, int cost, KvSegment& g) {
    while (x < x1) {
      if (!have) s = kv_seq<BM, TK>(r, page_log2, group, b), have = true;
      while (x - xb >= static_cast<int>(s.weight(heads, cost))) {  // ends: the sequences from b on reach beyond x < x1 <= W
        if (b + 1 >= r.B) return false;
        xb += s.weight(heads, cost);
        s = kv_seq<BM, TK>(r, page_log2, group, ++b);
      }
      const unsigned rem = x - xb, w = s.kt + cost, unit = rem / w;
      const int y = rem - unit * w, end = min(static_cast<int>(w), y + (x1 - x));
      g.s = s, g.b = b;
      g.k0 = max(0, y - cost), g.k1 = max(0, end - cost);
      g.x = x - y + cost;
      g.h = unit / static_cast<unsigned>(s.qt);
      g.u = unit - static_cast<unsigned>(g.h) * s.qt;
      x += end - y;
      if (g.k0 < g.k1) return true;
    }
    return false;
  }
};
// Keys that some row of row tile u sees: the last row's position + 1 (causal) or all of them.
template <int BM>
__device__ __forceinline__ int kv_visible(const KvSeq& s, int group, int u, bool causal) {
  if (!causal) return s.len;
  const int last = (min((u + 1) * BM, s.n * group) - 1) / group;
  return max(0, min(s.len, s.pos + last + 1));
}

// ---------------------------------------------------------------------------------------------
// TMA without a tensor map: a contiguous run of 16-byte units
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
inline bool kv_a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// the arguments every entry takes; 0 or an argument error. `what` names the entry.
int kv_fill_cache(KvCache* c, const char* what, const void* k, const void* v, const float* ks, const float* vs, int64_t pages,
                  int64_t heads, int64_t page, int64_t D, int fmt);
int kv_fill_rows(KvRows* r, const char* what, const int32_t* table, int64_t table_stride, int64_t per_seq, const int32_t* lens,
                 const int32_t* starts, int64_t B, int64_t T);

}  // namespace rh3
