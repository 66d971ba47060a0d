// What the grouped-query kernels share: the two activation types, and the step's rows as tokens of
// a paged cache (include/dsv41_b200.h, "Paged 8-bit KV cache").
#pragma once

#include "common.cuh"

namespace dsv41 {

// The activations' type as the kernels see it: bf16 or f16 values and pairs in registers.
template <bool F16>
struct Act;
template <>
struct Act<false> {
  using T = __nv_bfloat16;
  __device__ static float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  __device__ static uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  __device__ static float f(T x) { return __bfloat162float(x); }
  __device__ static T r(float x) { return __float2bfloat16_rn(x); }
};
template <>
struct Act<true> {
  using T = __half;
  __device__ static float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  __device__ static uint32_t pack(float lo, float hi) { return pack_f16x2(lo, hi); }
  __device__ static float f(T x) { return __half2float(x); }
  __device__ static T r(float x) { return __float2half_rn(x); }
};

// The step's rows and where their tokens lie.
struct StepRows {
  int T, seqs;
  const int* cu_rows;  // [seqs + 1], or null: row s is sequence s's only one
  const int* lens;     // [seqs]
  const int* table;    // [seqs, table_ld]
  int64_t table_ld;
  int width;           // table entries a sequence
};

struct KvCache {
  uint8_t *k, *v, *k_codes, *v_codes;
  int64_t pages;
  int kv_heads, page, block;
};

// The sequence of row r (a whole warp calls it; the same answer in every lane), or -1 for a row
// behind the last sequence: the number of ends cu_rows[1 ..] that are not past r.
__device__ __forceinline__ int row_seq(const StepRows& s, int r, int lane) {
  if (!s.cu_rows) return r;
  int n = 0;
  for (int i = 0; i < s.seqs; i += 32) {
    const bool before = i + lane < s.seqs && s.cu_rows[1 + i + lane] <= r;
    n += __popc(__ballot_sync(0xffffffffu, before));
  }
  return n < s.seqs && s.cu_rows[n] <= r ? n : -1;
}

// The page that holds token p >= 0 of sequence s, or -1 when there is none in range.
__device__ __forceinline__ int token_page(const StepRows& s, const KvCache& c, int seq, int p) {
  const int i = p / c.page;
  if (i >= s.width) return -1;
  const int pg = s.table[seq * s.table_ld + i];
  return pg >= 0 && pg < c.pages ? pg : -1;
}

}  // namespace dsv41
