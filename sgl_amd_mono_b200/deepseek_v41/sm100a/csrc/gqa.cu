// extern "C" entry points of the grouped-query decode operators (include/dsv41_b200.h): the 4-bit
// GEMV, the paged 8-bit cache's append and the attention over it. Argument checks, then the launches
// on the caller's stream.
#include <algorithm>
#include <climits>
#include <cstdio>
#include <cstring>
#include <type_traits>

#include "../../../../include/dsv41_b200.h"
#include "gemv_w4.cuh"
#include "gqa.cuh"
#include "kv_append.cuh"
#include "paged_attn.cuh"

using namespace dsv41;

namespace {

// Bytes of x that a CTA of the 4-bit GEMV keeps in shared memory; more is read through L1.
constexpr int64_t kW4XBytes = 40 * 1024;

template <class T>
T* ptr(int64_t v) {
  return reinterpret_cast<T*>(v);
}

// One launch with programmatic dependent launch (every kernel waits before it reads).
template <class Args>
int launch(void (*kernel)(const Args), dim3 grid, dim3 block, int smem, void* stream, const Args& args) {
  cudaError_t e = smem > 48 * 1024 ? ensure_smem(reinterpret_cast<const void*>(kernel), smem) : cudaSuccess;
  if (e == cudaSuccess) {
    count_launch();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_on() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, args);
  }
  if (e == cudaSuccess) return DSV41_OK;
  cudaGetLastError();
  fprintf(stderr, "dsv41: launch failed: %s\n", cudaGetErrorString(e));
  return DSV41_ELAUNCH;
}

int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows [T, heads, dim] of 2-byte values, ld elements apart.
bool rows_ok(int64_t p, int64_t ld, int64_t heads, int64_t dim) {
  return p && p % 16 == 0 && ld % 8 == 0 && ld >= heads * dim;
}

// What the append and the attention check alike: the cache's form and the step's rows.
template <class A>
bool paged_ok(const A* a) {
  return a && a->T >= 0 && a->T <= (1 << 24) && a->seqs >= 0 && a->seqs <= (1 << 20) && a->heads >= 1 &&
         a->heads <= 4096 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0 &&
         (a->dim == 64 || a->dim == 128 || a->dim == 256) && (a->f16 == 0 || a->f16 == 1) && a->lens &&
         a->lens % 4 == 0 && a->table && a->table % 4 == 0 && a->cu_rows % 4 == 0 && a->width >= 1 &&
         a->table_ld >= a->width && (a->cu_rows || a->T == a->seqs) && a->pages >= 1 && a->pages <= INT_MAX &&
         a->block >= 16 && a->block % 16 == 0 && a->page >= a->block && a->page <= (1 << 20) &&
         a->page % a->block == 0 && a->width <= INT_MAX / a->page && a->k_cache && a->v_cache &&
         a->k_cache % 16 == 0 && a->v_cache % 16 == 0 && a->k_codes && a->v_codes;
}

template <class A>
StepRows step_rows(const A* a) {
  return {(int)a->T, (int)a->seqs, ptr<const int>(a->cu_rows), ptr<const int>(a->lens), ptr<const int>(a->table),
          a->table_ld, (int)a->width};
}

template <class A>
KvCache kv_cache(const A* a) {
  return {ptr<uint8_t>(a->k_cache), ptr<uint8_t>(a->v_cache), ptr<uint8_t>(a->k_codes), ptr<uint8_t>(a->v_codes),
          a->pages, (int)a->kv_heads, (int)a->page, (int)a->block};
}

bool append_ok(const Dsv41KvAppendArgs* a) {
  return paged_ok(a) && rows_ok(a->k, a->k_ld, a->kv_heads, a->dim) && rows_ok(a->v, a->v_ld, a->kv_heads, a->dim) &&
         (!a->q || (rows_ok(a->q, a->q_ld, a->heads, a->dim) && rows_ok(a->q_out, a->q_out_ld, a->heads, a->dim))) &&
         a->rope >= 0 && a->rope <= a->dim && a->rope % 16 == 0 && (a->neox == 0 || a->neox == 1) &&
         (!a->rope || (a->cos_sin && a->cos_sin % 16 == 0 && a->rope_rows >= 1));
}

bool attn_ok(const Dsv41PagedAttnArgs* a) {
  return paged_ok(a) && rows_ok(a->q, a->q_ld, a->heads, a->dim) && rows_ok(a->out, a->out_ld, a->heads, a->dim) &&
         a->window >= 0 && a->window <= INT_MAX && a->sink % 4 == 0;
}

// Columns of 8 a CTA takes together. A sequence's columns (its rows times the query heads of a kv
// head; T / seqs rows on average) share every key that is read, so as many as they fill, up to the
// accumulators that fit: 32 columns of 64 or 128 dims, 16 of 256.
int attn_tiles(const Dsv41PagedAttnArgs* a) {
  const int64_t cols = a->heads / a->kv_heads * std::max<int64_t>(1, cdiv64(a->T, std::max<int64_t>(1, a->seqs)));
  return cols <= 8 ? 1 : cols <= 16 || a->dim == 256 ? 2 : 4;
}

template <int V>
using Int = std::integral_constant<int, V>;

// f(type, dim, column tiles) of the arguments' kernel.
template <class F>
int64_t attn_go(const Dsv41PagedAttnArgs* a, F f) {
  auto by_type = [&](auto d, auto nt) { return a->f16 ? f(Int<1>(), d, nt) : f(Int<0>(), d, nt); };
  auto by_tiles = [&](auto d) {
    switch (attn_tiles(a)) {
      case 1: return by_type(d, Int<1>());
      case 2: return by_type(d, Int<2>());
      default: return by_type(d, Int<d == 256 ? 2 : 4>());
    }
  };
  return a->dim == 64 ? by_tiles(Int<64>()) : a->dim == 128 ? by_tiles(Int<128>()) : by_tiles(Int<256>());
}

template <int D, int NT>
int64_t attn_ctas() {
  return (int64_t)device_sms() * PaShape<D, NT>::kCtas;
}
template <int D, int NT>
int64_t attn_scratch() {
  return 2 * attn_ctas<D, NT>() * 8 * NT * (D * sizeof(float) + sizeof(float4));
}

template <int F16, int D, int NT>
int attn_run(const Dsv41PagedAttnArgs* a, void* stream) {
  if (!a->scratch || a->scratch % 16 || a->scratch_bytes < attn_scratch<D, NT>()) return DSV41_ESCRATCH;
  const uint32_t bits = (uint32_t)a->scale_f32;
  float scale;
  memcpy(&scale, &bits, 4);
  const int64_t ctas = attn_ctas<D, NT>(), slots = 2 * ctas * 8 * NT;
  float* part = ptr<float>(a->scratch);
  const PagedAttnArgs p = {step_rows(a), kv_cache(a), (int)a->heads, (int)a->window, scale * 1.44269504f,
                           ptr<const void>(a->q), ptr<void>(a->out), a->q_ld, a->out_ld, ptr<const float>(a->sink),
                           part, reinterpret_cast<float4*>(part + slots * D)};
  const int rc = launch(paged_attn_kernel<F16, D, NT>, dim3((unsigned)ctas), dim3(32 * kPaWarps),
                        PaShape<D, NT>::kBytes, stream, p);
  return rc ? rc : launch(paged_join_kernel<F16, D, NT>, dim3((unsigned)ctas), dim3(32 * kPaWarps), 0, stream, p);
}

bool w4_ok(const Dsv41GemvW4Args* a) {
  return a && a->w && a->w % 16 == 0 && a->scales && a->scales % 2 == 0 && a->x && a->x % 16 == 0 && a->y &&
         a->y % 2 == 0 && a->M >= 1 && a->M <= kW4MaxRows && a->N >= 1 && a->N <= (1 << 24) && a->group >= 32 &&
         a->group % 32 == 0 && a->K >= a->group && a->K <= (1 << 24) && a->K % a->group == 0 && a->x_ld % 8 == 0 &&
         a->x_ld >= a->K && a->y_ld >= a->N && (a->f16 == 0 || a->f16 == 1);
}

template <int NT, int R, int GS>
int w4_run(int64_t f16, GemvW4Args g, void* stream) {
  using P = W4Shape<NT, R, GS>;
  // a lane's scales of a chunk in one load
  constexpr int el = P::kEntries > 1 ? P::kEntries / 2 : 1;
  g.vec = g.group == 32 * GS && g.K / g.group % el == 0 && g.K % kW4Chunk == 0 &&
          reinterpret_cast<uintptr_t>(g.scales) % (2 * el) == 0 && reinterpret_cast<uintptr_t>(g.zeros) % el == 0;
  const int64_t x_bytes = (int64_t)g.M * g.K * 2;
  const bool xs = x_bytes <= kW4XBytes;
  const int smem = P::kBytes + (xs ? (int)x_bytes : 0);
  // persistent: as many CTAs as fit, each taking every grid-th row tile
  const int fit = std::min(std::max(1, 226 * 1024 / (smem + 1024)), 4);
  const dim3 grid(std::min(cdiv(g.N, P::kRows), device_sms() * fit)), block(32 * kW4Warps);
  if (xs)
    return f16 ? launch(gemv_w4_kernel<true, NT, R, GS, true>, grid, block, smem, stream, g)
               : launch(gemv_w4_kernel<false, NT, R, GS, true>, grid, block, smem, stream, g);
  return f16 ? launch(gemv_w4_kernel<true, NT, R, GS, false>, grid, block, smem, stream, g)
             : launch(gemv_w4_kernel<false, NT, R, GS, false>, grid, block, smem, stream, g);
}

template <int NT, int R>
int w4_group(int64_t f16, const GemvW4Args& g, void* stream) {
  const int steps = g.group / 32;
  return steps % 8 == 0   ? w4_run<NT, R, 8>(f16, g, stream)
         : steps % 4 == 0 ? w4_run<NT, R, 4>(f16, g, stream)
         : steps % 2 == 0 ? w4_run<NT, R, 2>(f16, g, stream)
                          : w4_run<NT, R, 1>(f16, g, stream);
}

}  // namespace

extern "C" {

int dsv41_gemv_w4(const Dsv41GemvW4Args* a, void* stream) {
  if (!w4_ok(a)) return DSV41_EINVAL;
  GemvW4Args g = {ptr<const uint8_t>(a->w), ptr<const void>(a->scales), ptr<const uint8_t>(a->zeros),
                  ptr<const void>(a->x), ptr<void>(a->y), (int)a->M, (int)a->N, (int)a->K, (int)a->group,
                  a->x_ld, a->y_ld, 0};
  switch (cdiv(g.M, 8)) {
    // 32 weight rows a warp share a fragment of x; 16 make more work items of a small matrix (one row,
    // K 4096: N 4096 5.4 us with 16 and 5.6 with 32; N 8192 8.2 and 7.7; N 129280 79 and 69)
    case 1: return g.N >= 8192 ? w4_group<1, 2>(a->f16, g, stream) : w4_group<1, 1>(a->f16, g, stream);
    case 2: return w4_group<2, 2>(a->f16, g, stream);
    case 3: return w4_group<3, 2>(a->f16, g, stream);
    case 4: return w4_group<4, 2>(a->f16, g, stream);
    case 5: return w4_group<5, 2>(a->f16, g, stream);
    default: return w4_group<6, 2>(a->f16, g, stream);
  }
}

int dsv41_kv_append(const Dsv41KvAppendArgs* a, void* stream) {
  if (!append_ok(a)) return DSV41_EINVAL;
  if (!a->T || !a->seqs) return DSV41_OK;
  const KvAppendArgs k = {step_rows(a), kv_cache(a), (int)a->heads, (int)a->rope, (int)a->neox,
                          ptr<const void>(a->q), ptr<const void>(a->k), ptr<const void>(a->v), ptr<void>(a->q_out),
                          a->q_ld, a->q_out_ld, a->k_ld, a->v_ld, ptr<const float>(a->cos_sin), a->rope_rows};
  const int items = (a->q ? k.heads : 0) + 2 * k.cache.kv_heads;
  const dim3 grid(k.rows.T, cdiv(items, 4));
  switch (a->dim * 2 + a->f16) {
    case 128: return launch(kv_append_kernel<false, 64>, grid, dim3(128), 0, stream, k);
    case 129: return launch(kv_append_kernel<true, 64>, grid, dim3(128), 0, stream, k);
    case 256: return launch(kv_append_kernel<false, 128>, grid, dim3(128), 0, stream, k);
    case 257: return launch(kv_append_kernel<true, 128>, grid, dim3(128), 0, stream, k);
    case 512: return launch(kv_append_kernel<false, 256>, grid, dim3(128), 0, stream, k);
    default: return launch(kv_append_kernel<true, 256>, grid, dim3(128), 0, stream, k);
  }
}

int64_t dsv41_paged_attn_scratch_bytes(const Dsv41PagedAttnArgs* a) {
  if (!attn_ok(a)) return DSV41_EINVAL;
  return attn_go(a, [](auto, auto d, auto nt) { return attn_scratch<d, nt>(); });
}

int dsv41_paged_attn(const Dsv41PagedAttnArgs* a, void* stream) {
  if (!attn_ok(a)) return DSV41_EINVAL;
  if (!a->T || !a->seqs) return DSV41_OK;
  return (int)attn_go(a, [&](auto f16, auto d, auto nt) { return (int64_t)attn_run<f16, d, nt>(a, stream); });
}

}  // extern "C"
