// What the attention kernels over the quantized cache share: parameters, partial results and the numerics.
//
// For a query row i and cached token j:  t = scale * (q_i . kcode_j) * ks_j,  p = softmax_j(t),  o_i = sum_j p * vs_j * vcode_j.
// The scale of V goes into the exponent, so that the weights that meet the V codes are at most 1 whatever the scales are:
//     u_j = t_j * log2 e + log2 vs_j,   m = running max of u,   w_j = 2^(u_j - m + 15) in (0, 2^15]
//     l = sum w_j / vs_j,   O = sum fp16(w_j) * vcode_j,   o = O / l
// Codes are exact in fp16; q is scaled per row by a power of two into fp16 (exact for all but values 2^-28 below the row's
// largest); w is rounded to fp16 (2^-11 of the weight at most; bf16 would be 2^-8, as much as the rounding of the output), and the
// factor 2^15 keeps weights down to 2^-29 of the largest at that precision (normal numbers), so that the tail of a long context is not lost;
// products, sums, m, l and O are fp32. Partial results over parts of the keys carry (O, m, l) with the same m for both.
#pragma once
#include <atomic>
#include <limits>

#include "kv_cache.cuh"
#include "rapidh3_b200.h"

namespace rh3 {

struct KvAttnParams {
  KvCache c;
  KvRows r;
  const uint16_t* q;  // bf16 or fp16 [T][heads * group][D], strides below
  uint16_t* out;
  int64_t q_st, q_sh, o_st, o_sh;
  int is_f16;
  int group;          // query heads per KV head
  int causal;
  int cost;           // what a unit weighs besides its tiles
  float sl2;          // softmax scale * log2 e
  int* status;
  // partial results of units that more than one CTA works on: two slots per CTA (0: of the unit its run begins inside of, 1: of the unit
  // its run ends inside of)
  float* part;              // [grid][2][BM * D + 2 * BM]: O in fragment order, m, l
  int* count;               // [grid] parts written of the unit in a CTA's slot 1; all 0 between calls
  // shared prefix. Its pass writes every unit's parts row by row; the pass over the own keys takes them in.
  //   pre_o [split][heads][rows][D], pre_ml [split][heads][rows][2], rows = T * group
  float* pre_o;
  float* pre_ml;
  // which parts the prefix pass leaves of a unit, in its measure of work: a CTA has pre_run of it, a unit weighs pre_unit; the CTAs that
  // positions pre_first and pre_last of a unit belong to have its first and its last part
  int pre_run, pre_unit, pre_first, pre_last, pre_bm;
  // shared prefix in a single pass: r.pre_tiles tiles of it before a unit's own
  const int* pre_table;
  int pre_len;
};

// The slot of part i of a unit whose first tile is CTA `first`'s
__device__ __forceinline__ int64_t kv_slot(int first, int i) { return i == 0 ? 2ll * first + 1 : 2ll * (first + i); }

__device__ __forceinline__ float kv_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float kv_lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float kv_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The power of two that brings a row's largest magnitude to [2^14, 2^15), and its inverse (rows of zeros: 1).
__device__ __forceinline__ void kv_row_factor(float amax, float& up, float& down) {
  int e = static_cast<int>(__float_as_uint(amax) >> 23) & 0xFF;   // biased exponent
  e = max(e, 15);                                                 // both factors stay normal numbers
  up = amax > 0.f ? __uint_as_float(static_cast<uint32_t>(127 + 14 + 127 - e) << 23) : 1.f;
  down = amax > 0.f ? __uint_as_float(static_cast<uint32_t>(e - 14) << 23) : 1.f;
}
constexpr float kWeightLog2 = 15.f;   // the largest weight is 2^15: the most that fp16 holds as a power of two

// V scales as the kernels use them: a slot that was never written may hold 0
constexpr float kVsMin = 1e-30f;
// what makes a key's scores NaN, and so every row that sees it and no other
constexpr float kNan = std::numeric_limits<float>::quiet_NaN();

// Four codes of a word as two fp16 pairs: (byte 0, byte 1), (byte 2, byte 3), exactly.
template <int FMT>
__device__ __forceinline__ void kv_codes_to_half(uint32_t w, uint32_t& a, uint32_t& b) {
  if constexpr (FMT == RH3_KIND_I8) {
    // 0x64xx is 1024 + xx; xx = code + 128
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    uint32_t lo = __byte_perm(u, 0x64646464u, 0x4140), hi = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&lo), off), y = __hsub2(*reinterpret_cast<__half2*>(&hi), off);
    a = *reinterpret_cast<const uint32_t*>(&x);
    b = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(a) : "h"(static_cast<uint16_t>(w)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b) : "h"(static_cast<uint16_t>(w >> 16)));
  }
}

__device__ __forceinline__ float2 kv_unpack(uint32_t w, int is_f16) {
  if (is_f16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(bf16_lo(w), bf16_hi(w));
}
__device__ __forceinline__ uint32_t kv_pack(float a, float b, int is_f16) { return is_f16 ? pack_half2(a, b) : pack_bf16x2(a, b); }

// Lets `kern` have `smem` bytes of shared memory, once per device; `done` is the kernel's own word, a bit per device.
template <class K>
int kv_allow_smem(K kern, int smem, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (int e = check_cuda(cudaGetDevice(&dev), "kv_attn device")) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return 0;
  if (int e = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "kv_attn smem attribute")) return e;
  done.fetch_or(bit, std::memory_order_relaxed);
  return 0;
}

// kv_attn_wide.cu: the same parameters, units of 256 rows; floats of one of its partial results
constexpr int KV_WIDE_BM = 256;
// What a unit costs besides its keys, in keys: some 12 us of Q, first tile and output. (us with 256 / 512 / 640 / 1,024, 8 KV heads: 10 prompts of up to
// 512 x 4 rows behind 1,024 tokens 124 / 115 / 116 / 116, 37 fresh ones of up to 900 x 8 710 / 621 / 597 / 606, 4 of 1,500 x 4 183 / 168 / 169 / 178.)
constexpr int KV_WIDE_UNIT_COST = 640;
int64_t kv_wide_part_floats(int64_t D);
int kv_wide_launch(const KvAttnParams& p, int64_t D, int kind, bool prefix, int64_t grid, cudaStream_t stream);

}  // namespace rh3
