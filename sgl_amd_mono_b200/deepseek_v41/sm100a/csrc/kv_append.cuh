// Appending a step's keys and values to the paged e4m3 cache (dsv41_kv_append).
//
// Per block of `block` consecutive tokens of a head: code = code_ceil(max(amax, 1e-4) / 448) over
// the block's new tokens, at least the code of the older tokens in it; byte = e4m3(x 2^(127 -
// code)); when the code grows from c0 to c1, the older bytes become e4m3(byte 2^(c0 - c1)). The
// scale is a power of two, so only bytes that fall into e4m3's subnormal range change value.
// A block is written by one warp, that of its first new row, so no two warps meet in a block.
#pragma once

#include "gqa.cuh"

namespace dsv41 {

struct KvAppendArgs {
  StepRows rows;
  KvCache cache;
  int heads, rope, neox;
  const void *q, *k, *v;
  void* q_out;
  int64_t q_ld, q_out_ld, k_ld, v_ld;
  const float* cos_sin;
  int64_t rope_rows;
};

// e4m3 byte of x, saturating; NaN stays NaN.
__device__ __forceinline__ uint8_t kv_byte(float x) {
  return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

// Element d of a row's head, rotated when cs is not null: the pair's two products and their sum are
// each rounded in fp32, as the cache's contract says.
template <bool F16, int D>
__device__ __forceinline__ float rotated(const typename Act<F16>::T* x, int d, const float* cs, int rope, int neox) {
  const float v = Act<F16>::f(x[d]);
  const int i = d - (D - rope);
  if (!cs || i < 0) return v;
  const int half = rope / 2;
  const int pr = neox ? (i < half ? i : i - half) : i >> 1;
  const bool first = neox ? i < half : !(i & 1);
  const float o = Act<F16>::f(x[neox ? (first ? d + half : d - half) : (d ^ 1)]);
  const float c = cs[pr], s = cs[half + pr];
  return first ? __fsub_rn(__fmul_rn(v, c), __fmul_rn(o, s)) : __fadd_rn(__fmul_rn(o, s), __fmul_rn(v, c));
}

// Grid (T, ceil((heads + 2 kv_heads) / 4)), 128 threads: a warp a (row, head of q, k or v).
template <bool F16, int D>
__global__ void __launch_bounds__(128) kv_append_kernel(const KvAppendArgs a) {
  using T = typename Act<F16>::T;
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.x, kvh = a.cache.kv_heads;
  int h = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (!a.q) h += a.heads;
  if (h >= a.heads + 2 * kvh) return;
  const int seq = row_seq(a.rows, r, lane);
  if (seq < 0) return;
  const int first = a.rows.cu_rows ? a.rows.cu_rows[seq] : r;
  const int n = a.rows.cu_rows ? a.rows.cu_rows[seq + 1] - first : 1;
  const int64_t pos = (int64_t)a.rows.lens[seq] - n + (r - first);
  auto row_cs = [&](int64_t p) {
    return a.rope ? a.cos_sin + rope_row(max(p, (int64_t)0), a.rope_rows) * a.rope : nullptr;
  };
  if (h < a.heads) {
    const T* x = reinterpret_cast<const T*>(a.q) + r * a.q_ld + h * D;
    T* y = reinterpret_cast<T*>(a.q_out) + r * a.q_out_ld + h * D;
    const float* cs = row_cs(pos);
    float v[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) v[i] = rotated<F16, D>(x, lane + 32 * i, cs, a.rope, a.neox);
    __syncwarp();  // q_out may be q
#pragma unroll
    for (int i = 0; i < D / 32; ++i) y[lane + 32 * i] = Act<F16>::r(v[i]);
    return;
  }
  if (pos < 0 || pos >= (int64_t)a.rows.width * a.cache.page) return;
  const int block = a.cache.block, in = (int)(pos % block);
  if (r != first && in != 0) return;  // the warp of the block's first new row writes it
  const int pg = token_page(a.rows, a.cache, seq, (int)pos);
  if (pg < 0) return;
  const int off = (int)(pos % a.cache.page);
  const int rows = min(min(block - in, n - (r - first)), a.rows.T - r);
  const bool is_k = h < a.heads + kvh;
  const int hk = h - a.heads - (is_k ? 0 : kvh);
  const T* x = reinterpret_cast<const T*>(is_k ? a.k : a.v) + hk * D;
  const int64_t ld = is_k ? a.k_ld : a.v_ld;
  uint8_t* cache = is_k ? a.cache.k : a.cache.v;
  uint8_t* codes = is_k ? a.cache.k_codes : a.cache.v_codes;
  const int64_t head = (int64_t)pg * kvh + hk;
  uint8_t* dst = cache + (head * a.cache.page + off - in) * D;  // the block's first token
  uint8_t* cp = codes + head * (a.cache.page / block) + off / block;
  float amax = 0.f;
  for (int i = 0; i < rows; ++i)
    for (int d = lane; d < D; d += 32)
      amax = fmaxf(amax, fabsf(rotated<F16, D>(x + (r + i) * ld, d, is_k ? row_cs(pos + i) : nullptr, a.rope, a.neox)));
  amax = fminf(warp_max(amax), 3.402823466e38f);
  int code = code_ceil(__fdiv_rn(fmaxf(amax, 1e-4f), kFp8Max));
  if (in) {
    const int old = *cp;
    if (old >= code) code = old;
    else {
      const float m = pow2c(max(127 + old - code, 0));
      for (int i = lane; i < in * D; i += 32) dst[i] = kv_byte(e4m3_float(dst[i]) * m);
    }
  }
  const float mul = mx_mul(code);
  for (int i = 0; i < rows; ++i)
    for (int d = lane; d < D; d += 32)
      dst[(in + i) * D + d] =
          kv_byte(rotated<F16, D>(x + (r + i) * ld, d, is_k ? row_cs(pos + i) : nullptr, a.rope, a.neox) * mul);
  __syncwarp();
  if (lane == 0) *cp = (uint8_t)code;
}

}  // namespace dsv41
