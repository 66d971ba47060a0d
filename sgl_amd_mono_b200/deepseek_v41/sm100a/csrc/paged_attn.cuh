// Attention of decode and verify rows over the paged e4m3 cache (dsv41_paged_attn): per row and
// query head o = sum_i softmax(scale q . k_i)_i v_i over the keys the row sees, in one pass with the
// running maximum m and sum l of the softmax in fp32.
#pragma once

#include "gqa.cuh"

namespace dsv41 {

struct PagedAttnArgs {
  StepRows rows;
  KvCache cache;
  int heads, window;
  float scale;
  const void* q;
  void* out;
  int64_t q_ld, out_ld;
  const float* sink;  // [heads] or null
};

// Grid (T, ceil(heads / 4)), 128 threads: a warp a (row, query head), key by key.
template <bool F16, int D>
__global__ void __launch_bounds__(128) paged_attn_kernel(const PagedAttnArgs a) {
  using T = typename Act<F16>::T;
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (h >= a.heads) return;
  const int seq = row_seq(a.rows, r, lane);
  if (seq < 0) return;
  const int first = a.rows.cu_rows ? a.rows.cu_rows[seq] : r;
  const int n = a.rows.cu_rows ? a.rows.cu_rows[seq + 1] - first : 1;
  const int page = a.cache.page, block = a.cache.block, kvh = a.cache.kv_heads;
  const int vis = (int)min((int64_t)a.rows.lens[seq] - n + (r - first) + 1, (int64_t)a.rows.width * page);
  const int lo = a.window ? max(0, a.rows.lens[seq] - n + (r - first) + 1 - a.window) : 0;
  const int hk = h / (a.heads / kvh);
  const T* qp = reinterpret_cast<const T*>(a.q) + r * a.q_ld + h * D;
  float q[D / 32], o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) q[i] = Act<F16>::f(qp[lane + 32 * i]), o[i] = 0.f;
  float m = a.sink ? a.sink[h] : -INFINITY, l = a.sink ? 1.f : 0.f;
  for (int p = lo; p < vis; ++p) {
    const int pg = token_page(a.rows, a.cache, seq, p);
    if (pg < 0) continue;
    const int64_t head = (int64_t)pg * kvh + hk;
    const uint8_t* kp = a.cache.k + (head * page + p % page) * D;
    const uint8_t* vp = a.cache.v + (head * page + p % page) * D;
    const int64_t ci = head * (page / block) + p % page / block;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) s += q[i] * e4m3_float(kp[lane + 32 * i]);
    s = warp_sum(s) * pow2c(a.cache.k_codes[ci]) * a.scale;
    const float mn = fmaxf(m, s), f = m == mn ? 1.f : __expf(m - mn), w = __expf(s - mn);
    const float vs = w * pow2c(a.cache.v_codes[ci]);
    l = l * f + w;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = o[i] * f + vs * e4m3_float(vp[lane + 32 * i]);
    m = mn;
  }
  T* y = reinterpret_cast<T*>(a.out) + r * a.out_ld + h * D;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) y[lane + 32 * i] = Act<F16>::r(l == 0.f ? 0.f : o[i] / l);
}

}  // namespace dsv41
