// Writing rows into the quantized key/value cache and reading them back.
//
// A row is one token's D channels of one head. Written: s = max(amax / 127, 1e-12), code = rint(x / s) (int8), or
// s = max(amax / 448, 1e-12), code = e4m3(clamp(x / s)) -- the arithmetic of the row quantizers (quant.cu), codes and scales bit for bit.
// A row with a NaN or an infinity keeps it in its scale, its codes are 0: it reads back as NaN, and a masked one cannot reach
// a product through its codes. Read: code * s in fp32, rounded once to the asked type.
//
// HBM-bound copies: write takes in 2 * D * esize and puts out 2 * (D + 4) bytes per (token, head), read the reverse. A lane
// holds 8 channels (16-byte accesses on the bf16 side, 8 bytes on the code side), D / 8 lanes a row. A warp has KV_ITER groups of
// rows of one token, all of K or all of V, issues their loads before it works on the first, and looks up once where they lie
// (sequence, page); a block's eight warps have eight tokens, whose codes and scales of a head are neighbours in a page. Instructions are
// what such a warp has to save: its addresses are a pointer and a step, its token and part come from the grid. Measured, 36,436 tokens of
// 8 heads of 128 read as bf16, and 37 ragged prompts of up to 900 fp32 tokens written and read: 37 and 49 us, 93 and 90% of a copy's bandwidth
// (rows of K and V in one warp, an address per row and a division per warp, 471 instructions: 48.5 and 58 us; four tokens a warp
// besides: 84 and 69 us).
#include <cuda_bf16.h>

#include "kv_cache.cuh"
#include "rapidh3_b200.h"

namespace rh3 {
namespace {

constexpr int KV_THREADS = 256;
constexpr int KV_ITER = 4;

enum { KV_BF16 = 0, KV_F16 = 1, KV_F32 = 2 };

template <int DT>
struct KvRaw {  // eight elements of a row as loaded
  uint4 a, b;
};
template <int DT>
__device__ __forceinline__ void kv_load8(const void* base, int64_t at, KvRaw<DT>& r) {
  if constexpr (DT == KV_F32) {
    r.a = ld_global_16(static_cast<const float*>(base) + at);
    r.b = ld_global_16(static_cast<const float*>(base) + at + 4);
  } else {
    r.a = ld_global_16(static_cast<const uint16_t*>(base) + at);
  }
}
template <int DT>
__device__ __forceinline__ void kv_unpack8(const KvRaw<DT>& r, float* x) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
  if constexpr (DT == KV_F32) {
    const uint32_t u[4] = {r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(w[j]), x[4 + j] = __uint_as_float(u[j]);
  } else if constexpr (DT == KV_F16) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      x[2 * j] = f.x, x[2 * j + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[2 * j] = bf16_lo(w[j]), x[2 * j + 1] = bf16_hi(w[j]);
  }
}
// largest magnitude of the eight
template <int DT>
__device__ __forceinline__ float kv_amax8(const KvRaw<DT>& r) {
  if constexpr (DT == KV_F32) {
    float x[8];
    kv_unpack8<DT>(r, x);
    float a = fabsf(x[0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) a = max_nan(a, fabsf(x[j]));
    return a;
  } else {   // two at a time, as they are
    using T2 = std::conditional_t<DT == KV_F16, __half2, __nv_bfloat162>;
    const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
    T2 m = __habs2(*reinterpret_cast<const T2*>(&w[0]));
#pragma unroll
    for (int j = 1; j < 4; ++j) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const T2*>(&w[j])));
    return max_nan(__low2float(m), __high2float(m));
  }
}
// The codes of the row quantizers, of the quotients y / s rounded to fp32, without a division and without a branch: with inv = RN(1 / s) and q
// within an ulp of y / s, r = y - q * s is exact in an FMA and RN(q + r * inv) is the rounded quotient (Markstein, "Computation of elementary
// functions on the IBM RISC System/6000 processor", 1990). RN(y * inv) may be 1.5 ulp off, one such step brings it within an ulp. Nothing
// leaves the normal numbers where it matters: s is at least 1e-12 and at most 2^128 / 127, and quotients too small for that give the code 0 either way. (bf16 rows have quotients that lie exactly between two codes: dividing where the product lies near
// one, as the row quantizers do, sends a third of the warps down that path. 32 ragged prompts of up to 900 bf16 tokens to int8: 50 us that way, 43
// this.)
template <int FMT>
__device__ __forceinline__ uint2 kv_quant8(const float* y, float s, float inv) {
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float p = __fmul_rn(y[j], inv), near = __fmaf_rn(__fmaf_rn(-p, s, y[j]), inv, p);
    q[j] = __fmaf_rn(__fmaf_rn(-near, s, y[j]), inv, near);
    if constexpr (FMT == RH3_KIND_F8) q[j] = copysignf(q[j], y[j]);   // a zero keeps its sign
  }
  if constexpr (FMT == RH3_KIND_I8) {
    uint32_t t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = __float_as_uint(__fadd_rn(q[j], 12582912.f));   // the integer in the low bits
    return make_uint2(pack_low_bytes(t[0], t[1], t[2], t[3]), pack_low_bytes(t[4], t[5], t[6], t[7]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint16_t h;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(h) : "f"(q[2 * j]), "f"(q[2 * j + 1]));
      w[j] = h;
    }
    return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
  }
}

struct KvWriteParams {
  KvCache c;
  KvRows r;
  const void* k;
  const void* v;
  int64_t k_st, k_sh, v_st, v_sh;  // token and head strides in elements
  int* status;
};

// block (x, y): tokens 8 x .. 8 x + 7, a warp each; heads of part y / 2, of K (y even) or V
template <int D, int FMT, int DT>
__global__ void __launch_bounds__(KV_THREADS) kv_write_kernel(const KvWriteParams p) {
  constexpr int LANES = D / 8, ROWS = 32 / LANES;  // lanes per row, rows per pass of a warp
  grid_dependency_begin();
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (KV_THREADS / 32) + (threadIdx.x >> 5);
  if (t >= p.r.T) return;
  const bool is_v = blockIdx.y & 1;
  const int first = (blockIdx.y >> 1) * (KV_ITER * ROWS) + lane / LANES, ch = (lane % LANES) * 8;   // the lane's first head
  KvRaw<DT> raw[KV_ITER];
  {
    const int64_t step = is_v ? p.v_sh : p.k_sh;
    int64_t at = t * (is_v ? p.v_st : p.k_st) + first * step + ch;
#pragma unroll
    for (int i = 0; i < KV_ITER; ++i, at += ROWS * step) {
      raw[i].a = raw[i].b = make_uint4(0, 0, 0, 0);
      if (first + i * ROWS < p.c.heads) kv_load8<DT>(is_v ? p.v : p.k, at, raw[i]);
    }
  }
  bool known;
  const int64_t place = kv_place(p.c, p.r, static_cast<int>(t), lane, p.status, &known);
  if (place < 0) return;
  // Largest magnitudes: the lanes of a row halve what they carry while they exchange, so that lane l ends with that of group l % 4, whose scale
  // and inverse it works out for all (a butterfly and two divisions per group took 1.7 us more for the prompts above).
  static_assert(KV_ITER == 4, "a group for each of four neighbouring lanes");
  float a[KV_ITER];
#pragma unroll
  for (int i = 0; i < KV_ITER; ++i) a[i] = kv_amax8<DT>(raw[i]);
  const bool odd = lane & 1, high = lane & 2;
  const float a0 = max_nan(odd ? a[1] : a[0], __shfl_xor_sync(0xffffffffu, odd ? a[0] : a[1], 1));
  const float a1 = max_nan(odd ? a[3] : a[2], __shfl_xor_sync(0xffffffffu, odd ? a[2] : a[3], 1));
  float amax = max_nan(high ? a1 : a0, __shfl_xor_sync(0xffffffffu, high ? a0 : a1, 2));
#pragma unroll
  for (int o = 4; o < LANES; o <<= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  float s_own = __fdiv_rn(amax, FMT == RH3_KIND_I8 ? 127.f : 448.f);
  if (s_own < 1e-12f) s_own = 1e-12f;
  const float inv_own = __fdiv_rn(1.f, s_own);

  const int64_t at = place + (static_cast<int64_t>(first) << p.c.page_log2);
  const int mine = (lane & 3) * ROWS;
  if (lane % LANES < 4 && first + mine < p.c.heads) (is_v ? p.c.vs : p.c.ks)[at + (static_cast<int64_t>(mine) << p.c.page_log2)] = s_own;
  uint8_t* code = (is_v ? p.c.v : p.c.k) + at * D + ch;
#pragma unroll
  for (int i = 0; i < KV_ITER; ++i, code += (ROWS * D) << p.c.page_log2) {
    const float s = __shfl_sync(0xffffffffu, s_own, (lane & ~3) | i), inv = __shfl_sync(0xffffffffu, inv_own, (lane & ~3) | i);
    float x[8];
    kv_unpack8<DT>(raw[i], x);
    uint2 q = make_uint2(0, 0);
    if (s < INFINITY) q = kv_quant8<FMT>(x, s, inv);
    if (first + i * ROWS < p.c.heads) *reinterpret_cast<uint2*>(code) = q;
  }
}

struct KvReadParams {
  KvCache c;
  KvRows r;
  void* k;
  void* v;  // [T][heads][D], contiguous
  int* status;
};

template <int FMT>
__device__ __forceinline__ void kv_decode8(uint2 q, float s, float* x) {
  const uint32_t w[2] = {q.x, q.y};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if constexpr (FMT == RH3_KIND_I8) {
      // the byte behind 2^23 is a float: 2^23 + (code + 128), exactly
      const uint32_t u = w[j] ^ 0x80808080u;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        x[4 * j + b] = __fmul_rn(__fsub_rn(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + b)), 8388736.f), s);
    } else {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t h2;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(w[j] >> (16 * b))));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
        x[4 * j + 2 * b] = __fmul_rn(f.x, s), x[4 * j + 2 * b + 1] = __fmul_rn(f.y, s);
      }
    }
  }
}

// blocks as kv_write_kernel's
template <int D, int FMT, int DT>
__global__ void __launch_bounds__(KV_THREADS) kv_read_kernel(const KvReadParams p) {
  constexpr int LANES = D / 8, ROWS = 32 / LANES;
  grid_dependency_begin();
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (KV_THREADS / 32) + (threadIdx.x >> 5);
  if (t >= p.r.T) return;
  const bool is_v = blockIdx.y & 1;
  const int first = (blockIdx.y >> 1) * (KV_ITER * ROWS) + lane / LANES, ch = (lane % LANES) * 8;
  bool known;
  const int64_t place = kv_place(p.c, p.r, static_cast<int>(t), lane, p.status, &known);
  if (!known) return;  // rows behind the last sequence stay as they are
  uint2 q[KV_ITER];
  float s[KV_ITER];
  {
    const int64_t at = place + (static_cast<int64_t>(first) << p.c.page_log2);
    const uint8_t* code = (is_v ? p.c.v : p.c.k) + at * D + ch;
    const float* scale = (is_v ? p.c.vs : p.c.ks) + at;
#pragma unroll
    for (int i = 0; i < KV_ITER; ++i, code += (ROWS * D) << p.c.page_log2, scale += ROWS << p.c.page_log2) {
      q[i] = make_uint2(0, 0);
      s[i] = 0.f;
      if (place >= 0 && first + i * ROWS < p.c.heads) {
        q[i] = *reinterpret_cast<const uint2*>(code);
        s[i] = *scale;
      }
    }
  }
  const int64_t to = (t * p.c.heads + first) * D + ch;
#pragma unroll
  for (int i = 0; i < KV_ITER; ++i) {
    if (first + i * ROWS >= p.c.heads) break;
    float x[8];
    kv_decode8<FMT>(q[i], s[i], x);
    if constexpr (DT == KV_F32) {
      float4* o = reinterpret_cast<float4*>(static_cast<float*>(is_v ? p.v : p.k) + to + i * ROWS * D);
      o[0] = make_float4(x[0], x[1], x[2], x[3]);
      o[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      uint32_t u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (DT == KV_F16) {
          const __half2 h = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
          u[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          u[j] = pack_bf16x2(x[2 * j], x[2 * j + 1]);
        }
      }
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(is_v ? p.v : p.k) + to + i * ROWS * D) = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
}

// calls fn(D, FMT, DT) as compile-time constants
template <class F>
int kv_dispatch(int64_t D, int fmt, int dt, F&& fn) {
  auto by_type = [&](auto d, auto f) {
    switch (dt) {
      case KV_BF16: return fn(d, f, std::integral_constant<int, KV_BF16>());
      case KV_F16: return fn(d, f, std::integral_constant<int, KV_F16>());
      default: return fn(d, f, std::integral_constant<int, KV_F32>());
    }
  };
  auto by_fmt = [&](auto d) {
    return fmt == RH3_KIND_I8 ? by_type(d, std::integral_constant<int, RH3_KIND_I8>())
                              : by_type(d, std::integral_constant<int, RH3_KIND_F8>());
  };
  return D == 64 ? by_fmt(std::integral_constant<int, 64>()) : by_fmt(std::integral_constant<int, 128>());
}

dim3 kv_grid(int64_t T, int64_t heads, int64_t D) {
  const int64_t rows = 32 / (D / 8) * KV_ITER;
  return dim3(static_cast<unsigned>((T + KV_THREADS / 32 - 1) / (KV_THREADS / 32)), static_cast<unsigned>(2 * ((heads + rows - 1) / rows)));
}

}  // namespace

int kv_fill_cache(KvCache* c, const char* what, const void* k, const void* v, const float* ks, const float* vs, int64_t pages,
                  int64_t heads, int64_t page, int64_t D, int fmt) {
  RH3_CHECK_ARG(fmt == RH3_KIND_I8 || fmt == RH3_KIND_F8, "%s: kind=%d must be 0 (int8) or 1 (e4m3)", what, fmt);
  RH3_CHECK_ARG(D == 64 || D == 128, "%s: head size %lld must be 64 or 128", what, (long long)D);
  RH3_CHECK_ARG(page == 16 || page == 32 || page == 64 || page == 128, "%s: pages of %lld tokens: must be 16, 32, 64 or 128", what,
                (long long)page);
  RH3_CHECK_ARG(heads > 0 && heads <= 1024 && pages > 0, "%s: bad cache shape: %lld pages, %lld heads", what, (long long)pages,
                (long long)heads);
  // TMA coordinates count rows of 128 bytes in 32 bits
  RH3_CHECK_ARG(pages <= (1ll << 31) / (heads * page * D / 128) - 1, "%s: a cache of %lld pages is too large", what, (long long)pages);
  RH3_CHECK_ARG(k && v && ks && vs && kv_a16(k) && kv_a16(v) && kv_a16(ks) && kv_a16(vs),
                "%s: cache pointers must be set and 16-byte aligned", what);
  c->k = static_cast<uint8_t*>(const_cast<void*>(k));
  c->v = static_cast<uint8_t*>(const_cast<void*>(v));
  c->ks = const_cast<float*>(ks);
  c->vs = const_cast<float*>(vs);
  c->pages = static_cast<int>(pages);
  c->heads = static_cast<int>(heads);
  c->page_log2 = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7;
  return 0;
}

int kv_fill_rows(KvRows* r, const char* what, const int32_t* table, int64_t table_stride, int64_t per_seq, const int32_t* lens,
                 const int32_t* starts, int64_t B, int64_t T) {
  RH3_CHECK_ARG(B > 0 && B <= 65536 && per_seq >= 0 && per_seq < (1 << 24) && table_stride >= per_seq,
                "%s: bad batch: %lld sequences, %lld pages each, stride %lld", what, (long long)B, (long long)per_seq,
                (long long)table_stride);
  RH3_CHECK_ARG(T >= 0 && T < (1 << 26), "%s: %lld rows: must be below 2^26", what, (long long)T);
  RH3_CHECK_ARG((table || per_seq == 0) && lens && starts, "%s: null batch pointer", what);
  *r = KvRows{table, lens, starts, table_stride, static_cast<int>(B), static_cast<int>(per_seq), static_cast<int>(T), 0, 0};
  return 0;
}

}  // namespace rh3

using namespace rh3;

extern "C" int rh3_kv_write(const rh3_kv_rows_args* a, cudaStream_t stream) {
  RH3_CHECK_ARG(a, "kv_write: null arguments");
  KvWriteParams p{};
  RH3_CHECK_ARG(a->dtype >= 0 && a->dtype <= 2, "kv_write: dtype=%d must be 0 (bf16), 1 (fp16) or 2 (fp32)", a->dtype);
  if (int e = kv_fill_cache(&p.c, "kv_write", a->kc, a->vc, a->ks, a->vs, a->pages, a->heads, a->page, a->D, a->kind)) return e;
  if (int e = kv_fill_rows(&p.r, "kv_write", a->table, a->table_stride, a->per_seq, a->lens, a->starts, a->B, a->T)) return e;
  if (a->T == 0) return 0;
  const int64_t per16 = a->dtype == KV_F32 ? 4 : 8;
  RH3_CHECK_ARG(a->k && a->v && kv_a16(a->k) && kv_a16(a->v) && a->k_st % per16 == 0 && a->k_sh % per16 == 0 && a->v_st % per16 == 0 && a->v_sh % per16 == 0,
                "kv_write: every row of k and v must start on a 16-byte boundary");
  p.k = a->k, p.v = a->v, p.k_st = a->k_st, p.k_sh = a->k_sh, p.v_st = a->v_st, p.v_sh = a->v_sh;
  p.status = device_status_word();
  const dim3 grid = kv_grid(a->T, a->heads, a->D);
  const bool chained = static_cast<int64_t>(grid.x) * grid.y <= 4 * device_sm_count() && !in_capture(stream);
  return kv_dispatch(a->D, a->kind, a->dtype, [&](auto d, auto f, auto t) {
    return check_cuda(launch_kernel(chained, kv_write_kernel<d(), f(), t()>, grid, KV_THREADS, 0, stream, 1, p),
                      "kv_write launch");
  });
}

extern "C" int rh3_kv_read(const rh3_kv_rows_args* a, cudaStream_t stream) {
  RH3_CHECK_ARG(a, "kv_read: null arguments");
  KvReadParams p{};
  RH3_CHECK_ARG(a->dtype >= 0 && a->dtype <= 2, "kv_read: dtype=%d must be 0 (bf16), 1 (fp16) or 2 (fp32)", a->dtype);
  if (int e = kv_fill_cache(&p.c, "kv_read", a->kc, a->vc, a->ks, a->vs, a->pages, a->heads, a->page, a->D, a->kind)) return e;
  if (int e = kv_fill_rows(&p.r, "kv_read", a->table, a->table_stride, a->per_seq, a->lens, a->starts, a->B, a->T)) return e;
  if (a->T == 0) return 0;
  RH3_CHECK_ARG(a->k && a->v && kv_a16(a->k) && kv_a16(a->v), "kv_read: outputs must be set and 16-byte aligned");
  p.k = a->k, p.v = a->v;
  p.status = device_status_word();
  const dim3 grid = kv_grid(a->T, a->heads, a->D);
  const bool chained = static_cast<int64_t>(grid.x) * grid.y <= 4 * device_sm_count() && !in_capture(stream);
  return kv_dispatch(a->D, a->kind, a->dtype, [&](auto d, auto f, auto t) {
    return check_cuda(launch_kernel(chained, kv_read_kernel<d(), f(), t()>, grid, KV_THREADS, 0, stream, 1, p),
                      "kv_read launch");
  });
}
