// extern "C" entry points of the grouped-query decode operators (include/dsv41_b200.h): the 4-bit
// GEMV, the paged 8-bit cache's append and the attention over it. Argument checks, then the launches
// on the caller's stream.
#include <climits>
#include <cstdio>
#include <cstring>

#include "../../../../include/dsv41_b200.h"
#include "gemv_w4.cuh"
#include "gqa.cuh"
#include "kv_append.cuh"
#include "paged_attn.cuh"

using namespace dsv41;

namespace {

template <class T>
T* ptr(int64_t v) {
  return reinterpret_cast<T*>(v);
}

template <class Args>
int launch(void (*kernel)(const Args), dim3 grid, dim3 block, int smem, void* stream, const Args& args) {
  count_launch();
  kernel<<<grid, block, smem, reinterpret_cast<cudaStream_t>(stream)>>>(args);
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return DSV41_OK;
  fprintf(stderr, "dsv41: launch failed: %s\n", cudaGetErrorString(e));
  return DSV41_ELAUNCH;
}

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

bool w4_ok(const Dsv41GemvW4Args* a) {
  return a && a->w && a->w % 16 == 0 && a->scales && a->scales % 2 == 0 && a->x && a->x % 16 == 0 && a->y &&
         a->y % 2 == 0 && a->M >= 1 && a->M <= kW4MaxRows && a->N >= 1 && a->N <= (1 << 24) && a->group >= 32 &&
         a->group % 32 == 0 && a->K >= a->group && a->K <= (1 << 24) && a->K % a->group == 0 && a->x_ld % 8 == 0 &&
         a->x_ld >= a->K && a->y_ld >= a->N && (a->f16 == 0 || a->f16 == 1);
}

}  // namespace

extern "C" {

int dsv41_gemv_w4(const Dsv41GemvW4Args* a, void* stream) {
  if (!w4_ok(a)) return DSV41_EINVAL;
  const GemvW4Args g = {ptr<const uint8_t>(a->w), ptr<const void>(a->scales), ptr<const uint8_t>(a->zeros),
                        ptr<const void>(a->x), ptr<void>(a->y), (int)a->M, (int)a->N, (int)a->K, (int)a->group,
                        a->x_ld, a->y_ld};
  return launch(a->f16 ? gemv_w4_kernel<true> : gemv_w4_kernel<false>, dim3(cdiv(g.N, 8)), dim3(256), 0, stream, g);
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

int64_t dsv41_paged_attn_scratch_bytes(const Dsv41PagedAttnArgs* a) { return attn_ok(a) ? 0 : DSV41_EINVAL; }

int dsv41_paged_attn(const Dsv41PagedAttnArgs* a, void* stream) {
  if (!attn_ok(a)) return DSV41_EINVAL;
  if (!a->T || !a->seqs) return DSV41_OK;
  const uint32_t bits = (uint32_t)a->scale_f32;
  float scale;
  memcpy(&scale, &bits, 4);
  const PagedAttnArgs p = {step_rows(a), kv_cache(a), (int)a->heads, (int)a->window, scale, ptr<const void>(a->q),
                           ptr<void>(a->out), a->q_ld, a->out_ld, ptr<const float>(a->sink)};
  const dim3 grid(p.rows.T, cdiv(p.heads, 4));
  switch (a->dim * 2 + a->f16) {
    case 128: return launch(paged_attn_kernel<false, 64>, grid, dim3(128), 0, stream, p);
    case 129: return launch(paged_attn_kernel<true, 64>, grid, dim3(128), 0, stream, p);
    case 256: return launch(paged_attn_kernel<false, 128>, grid, dim3(128), 0, stream, p);
    case 257: return launch(paged_attn_kernel<true, 128>, grid, dim3(128), 0, stream, p);
    case 512: return launch(paged_attn_kernel<false, 256>, grid, dim3(128), 0, stream, p);
    default: return launch(paged_attn_kernel<true, 256>, grid, dim3(128), 0, stream, p);
  }
}

}  // extern "C"
