// Appending a step's keys and values to the paged e4m3 cache (dsv41_kv_append).
//
// Per block of `block` consecutive tokens of a head: code = code_ceil(max(amax, 1e-4) / 448) over
// the block's new tokens, at least the code of the older tokens in it; byte = e4m3(x 2^(127 -
// code)); when the code grows from c0 to c1, the older bytes become e4m3(byte 2^(c0 - c1)). The
// scale is a power of two, so only bytes that fall into e4m3's subnormal range change value.
// A block is written by one warp, that of its first new row, so no two warps meet in a block.
//
// The work is copying, so everything moves 16 bytes a lane at a time in units of 16 dims: two 8-dim
// pieces that hold 8 whole rotation pairs and share 8 angles, side by side for pairs (2j, 2j + 1) and
// half a rotation apart for (j, j + rope / 2). A block's rows are looked at twice, for the largest
// magnitude and to be written, some of them in registers and the others from L1.
//
// One token 3.1 us and 8 sequences of 6 rows 3.6: dependent latencies (row, length, page, code). Prompts of
// 10266 rows, 32 query and 8 kv heads of 128: 48 us (4.9 TB/s of 236 MB). The queries alone take 29 us, a copy of
// them 27; the keys and values 23, which is latency and the second look, not bytes (10 us). Four CTAs an SM leave
// 64 registers a thread, of which every instance spills some (60 bytes reloaded with pairs side by side, 128
// half a rotation apart); fewer CTAs were slower (59 us to 53 when that was measured).
#pragma once

#include "gqa.cuh"

namespace dsv41 {

constexpr int kApThreads = 256;

struct KvAppendArgs {
  StepRows rows;
  KvCache cache;
  int heads, rope;
  const void *q, *k, *v;
  void* q_out;
  int64_t q_ld, q_out_ld, k_ld, v_ld;
  const float* cos_sin;
  int64_t rope_rows;
  int window;     // rows a warp looks through for blocks to write
  int kv_ctas;    // CTAs of the keys and values; the rest rotate queries
  int head_step;  // heads a query thread takes
};

// Dims of unit u of a head: its two pieces of 8, and the first of its 8 angles (< 0: not rotated).
struct RopeUnit {
  int d0, d1, angle;
};
template <bool NEOX>
__device__ __forceinline__ RopeUnit rope_unit(int u, int dim, int rope) {
  const int ur = u - (dim - rope) / 16;
  if (NEOX && ur >= 0) return {dim - rope + 8 * ur, dim - rope / 2 + 8 * ur, 8 * ur};
  return {16 * u, 16 * u + 8, ur >= 0 ? 8 * ur : -1};
}

template <bool F16>
__device__ __forceinline__ void unpack8(uint4 w, float* v) {
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Act<F16>::unpack(ws[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
struct Angles {
  float c[8], s[8];
};
__device__ __forceinline__ void load_angles(const float* row, int rope, int angle, Angles& a) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 c = __ldg(reinterpret_cast<const float4*>(row + angle) + i);
    const float4 s = __ldg(reinterpret_cast<const float4*>(row + rope / 2 + angle) + i);
    a.c[4 * i] = c.x, a.c[4 * i + 1] = c.y, a.c[4 * i + 2] = c.z, a.c[4 * i + 3] = c.w;
    a.s[4 * i] = s.x, a.s[4 * i + 1] = s.y, a.s[4 * i + 2] = s.z, a.s[4 * i + 3] = s.w;
  }
}
// The pair's two products and their sum are each rounded in fp32, as the cache's contract says.
__device__ __forceinline__ void rotate_pair(float& x, float& y, float c, float s) {
  const float a = x, b = y;
  x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  y = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
}
template <bool NEOX>
__device__ __forceinline__ void rotate16(float (&v)[16], const Angles& a) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (NEOX) rotate_pair(v[i], v[8 + i], a.c[i], a.s[i]);
    else rotate_pair(v[2 * i], v[2 * i + 1], a.c[i], a.s[i]);
  }
}
// 4 e4m3 bytes, saturating; NaN stays NaN.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

// The rows [r, r + rows) of one head, tokens `pos` .. of one block (its `in`th token on), by one warp.
template <bool F16, int D, bool NEOX>
__device__ __forceinline__ void append_block(const KvAppendArgs& a, int seq, int r, int rows, int pos, int in, int item) {
  using T = typename Act<F16>::T;
  constexpr int UNITS = D / 16, PER = 32 / UNITS;  // lanes a row, rows at a time
  const int lane = threadIdx.x & 31, kvh = a.cache.kv_heads, block = a.cache.block, page = a.cache.page;
  const int pg = token_page(a.rows, a.cache, seq, pos);
  if (pg < 0) return;
  const bool is_k = item < kvh;
  const int hk = is_k ? item : item - kvh;
  const int off = pos % page - in;  // the block's first token in its page
  const T* x = reinterpret_cast<const T*>(is_k ? a.k : a.v) + hk * D;
  const int64_t ld = is_k ? a.k_ld : a.v_ld;
  const int64_t head = (int64_t)pg * kvh + hk;
  uint8_t* dst = (is_k ? a.cache.k : a.cache.v) + (head * page + off) * D;
  uint8_t* cp = (is_k ? a.cache.k_codes : a.cache.v_codes) + head * (page / block) + off / block;
  const int rope = is_k ? a.rope : 0;
  const RopeUnit ru = rope_unit<NEOX>(lane % UNITS, D, rope);
  const int old = in ? *cp : 0;
  // the lane's units of rows i, i + PER, ..: the first KEEP stay in registers for the second pass, the others
  // come from L1 again (ragged prompts: 1 47.4 us, 2 48.9, 4 over 59 at the two CTAs an SM that it leaves)
  constexpr int KEEP = 1;
  auto load = [&](int i, uint4 (&w)[2]) {
    const T* row = x + (r + i) * ld;
    w[0] = ldg16(row + ru.d0);
    w[1] = ldg16(row + ru.d1);
  };
  auto value = [&](int i, const uint4 (&w)[2], float (&v)[16]) {
    unpack8<F16>(w[0], v);
    unpack8<F16>(w[1], v + 8);
    if (rope && ru.angle >= 0) {
      Angles an;
      load_angles(a.cos_sin + rope_row(pos + i, a.rope_rows) * rope, rope, ru.angle, an);
      rotate16<NEOX>(v, an);
    }
  };
  const int i0 = lane / UNITS;
  uint4 kept[KEEP][2];
#pragma unroll
  for (int n = 0; n < KEEP; ++n)
    if (i0 + n * PER < rows) load(i0 + n * PER, kept[n]);
  float amax = 0.f;
  auto see = [&](int i, const uint4 (&w)[2]) {
    float v[16];
    value(i, w, v);
#pragma unroll
    for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(v[e]));  // NaN does not count
  };
#pragma unroll
  for (int n = 0; n < KEEP; ++n)
    if (i0 + n * PER < rows) see(i0 + n * PER, kept[n]);
  for (int i = i0 + KEEP * PER; i < rows; i += PER) {
    uint4 w[2];
    load(i, w);
    see(i, w);
  }
  amax = fminf(warp_max(amax), 3.402823466e38f);
  int code = code_ceil(__fdiv_rn(fmaxf(amax, 1e-4f), kFp8Max));
  if (in) {
    if (old >= code) {
      code = old;
    } else {
      const float m = pow2c(max(127 + old - code, 0));
      uint32_t* w = reinterpret_cast<uint32_t*>(dst);
      for (int i = lane; i < in * (D / 4); i += 32) {
        const uint32_t b = w[i];
        const float2 lo = e4m3x2_float2(b & 0xffff), hi = e4m3x2_float2(b >> 16);
        w[i] = e4m3x4(lo.x * m, lo.y * m, hi.x * m, hi.y * m);
      }
    }
  }
  const float mul = mx_mul(code);
  auto put = [&](int i, const uint4 (&x)[2]) {
    float v[16];
    value(i, x, v);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = e4m3x4(v[4 * e] * mul, v[4 * e + 1] * mul, v[4 * e + 2] * mul, v[4 * e + 3] * mul);
    uint8_t* y = dst + (in + i) * D;
    *reinterpret_cast<uint2*>(y + ru.d0) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(y + ru.d1) = make_uint2(w[2], w[3]);
  };
#pragma unroll
  for (int n = 0; n < KEEP; ++n)
    if (i0 + n * PER < rows) put(i0 + n * PER, kept[n]);
  for (int i = i0 + KEEP * PER; i < rows; i += PER) {
    uint4 w[2];
    load(i, w);
    put(i, w);
  }
  __syncwarp();
  if (lane == 0) *cp = (uint8_t)code;
}

// The sequence of row r by binary search, or -1 for a row behind the last sequence.
__device__ __forceinline__ int row_seq_search(const StepRows& s, int r) {
  if (!s.cu_rows) return r;
  int lo = 0, hi = s.seqs;  // the first sequence whose end is past r
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (__ldg(s.cu_rows + mid + 1) > r) hi = mid;
    else lo = mid + 1;
  }
  return lo < s.seqs && __ldg(s.cu_rows + lo) <= r ? lo : -1;
}

// CTAs [0, kv_ctas): a warp a (window of rows, key or value head); the others: a thread a (row, head_step
// query heads, unit).
template <bool F16, int D, bool NEOX>
__global__ void __launch_bounds__(kApThreads, 4) kv_append_kernel(const KvAppendArgs a) {
  using T = typename Act<F16>::T;
  constexpr int UNITS = D / 16;
  pdl_wait();
  const StepRows& st = a.rows;
  if ((int)blockIdx.x < a.kv_ctas) {
    const int lane = threadIdx.x & 31, items = 2 * a.cache.kv_heads, block = a.cache.block;
    const uint32_t wi = blockIdx.x * (kApThreads / 32) + (threadIdx.x >> 5), window = wi / items;
    const int64_t w0 = (int64_t)window * a.window;
    if (w0 >= st.T) return;
    const int item = wi - window * items, w1 = (int)min(w0 + a.window, (int64_t)st.T);
    const int64_t cap = (int64_t)st.width * a.cache.page;
    int r = (int)w0, seq = row_seq(st, r, lane);
    while (r < w1 && seq >= 0 && seq < st.seqs) {
      const int first = st.cu_rows ? st.cu_rows[seq] : seq, end = st.cu_rows ? st.cu_rows[seq + 1] : seq + 1;
      if (end <= r) {
        ++seq;
        continue;
      }
      const int64_t pos = (int64_t)st.lens[seq] - end + r;
      int rows = end - r;  // to the next block's first row, or the sequence's end
      if (pos < 0) {
        rows = (int)min((int64_t)rows, -pos);
      } else {
        const int in = (uint32_t)pos % block;  // pos < lens[seq]
        rows = min(min(rows, block - in), st.T - r);
        // the block's first new row leads: the sequence's first, one at the block's start, or token 0
        if ((r == first || !in) && pos < cap) append_block<F16, D, NEOX>(a, seq, r, rows, (int)pos, in, item);
      }
      r += rows;
    }
    return;
  }
  const int groups = (a.heads + a.head_step - 1) / a.head_step;
  const uint32_t ti = (blockIdx.x - a.kv_ctas) * kApThreads + threadIdx.x, per = groups * UNITS;
  const int64_t row = ti / per;
  if (row >= st.T) return;
  const int r = (int)row, u = ti % UNITS, h0 = (ti - (uint32_t)r * per) / UNITS * a.head_step;
  const RopeUnit ru = rope_unit<NEOX>(u, D, a.rope);
  const T* x = reinterpret_cast<const T*>(a.q) + row * a.q_ld;
  // Every load ahead of the first store and of the search for the sequence (plain loads: the queries may be
  // rotated in place, a thread's own values each).
  constexpr int HEADS = 4;
  uint4 in[HEADS][2];
#pragma unroll
  for (int n = 0; n < HEADS; ++n)
    if (n < a.head_step && h0 + n < a.heads) {
      in[n][0] = *reinterpret_cast<const uint4*>(x + (h0 + n) * D + ru.d0);
      in[n][1] = *reinterpret_cast<const uint4*>(x + (h0 + n) * D + ru.d1);
    }
  const int seq = row_seq_search(st, r);
  if (seq < 0) return;
  Angles an;
  if (a.rope && ru.angle >= 0) {
    const int64_t pos = (int64_t)st.lens[seq] - (st.cu_rows ? st.cu_rows[seq + 1] : seq + 1) + r;
    load_angles(a.cos_sin + rope_row(max(pos, (int64_t)0), a.rope_rows) * a.rope, a.rope, ru.angle, an);
  }
  T* y = reinterpret_cast<T*>(a.q_out) + row * a.q_out_ld;
#pragma unroll
  for (int n = 0; n < HEADS; ++n)
    if (n < a.head_step && h0 + n < a.heads) {
      float v[16];
      unpack8<F16>(in[n][0], v);
      unpack8<F16>(in[n][1], v + 8);
      if (a.rope && ru.angle >= 0) rotate16<NEOX>(v, an);
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = Act<F16>::pack(v[2 * e], v[2 * e + 1]);
      *reinterpret_cast<uint4*>(y + (h0 + n) * D + ru.d0) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(y + (h0 + n) * D + ru.d1) = make_uint4(w[4], w[5], w[6], w[7]);
    }
}

}  // namespace dsv41
