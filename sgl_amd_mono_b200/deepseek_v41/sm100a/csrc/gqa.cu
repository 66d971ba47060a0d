// extern "C" entry points of the paged 8-bit cache's append and the attention over it
// (include/dsv41_b200.h): argument checks, then the launches on the caller's stream.
#include <algorithm>
#include <climits>
#include <cstring>
#include <numeric>
#include <type_traits>

#include "../../../../include/dsv41_b200.h"
#include "gqa.cuh"
#include "gqa_launch.cuh"
#include "kv_append.cuh"
#include "paged_attn.cuh"

using namespace dsv41;

namespace {

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
         a->window >= 0 && a->window <= INT_MAX && a->sink % 4 == 0 && a->T * (a->heads / a->kv_heads) <= (1 << 30);
}

// Columns of 8 a CTA takes together. A sequence's columns (its rows times the query heads of a kv
// head; T / seqs rows on average) share every key that is read, so as many as they fill, up to the
// accumulators that fit: 32 columns of 64 or 128 dims, 16 of 256.
int attn_tiles(const Dsv41PagedAttnArgs* a) {
  const int64_t cols = a->heads / a->kv_heads * std::max<int64_t>(1, cdiv64(a->T, std::max<int64_t>(1, a->seqs)));
  return cols <= 8 ? 1 : cols <= 16 || a->dim == 256 ? 2 : cols <= 24 ? 3 : 4;
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
      case 3: return by_type(d, Int<d == 256 ? 2 : 3>());
      default: return by_type(d, Int<d == 256 ? 2 : 4>());
    }
  };
  return a->dim == 64 ? by_tiles(Int<64>()) : a->dim == 128 ? by_tiles(Int<128>()) : by_tiles(Int<256>());
}

// How the work is cut, from what the host knows: the pages that the table can name and the window bound the
// steps of an item, the rows the items. Whole items, a CTA each, take one launch and no scratch; or the
// GPU's CTAs share all steps, no more of them than there can be, and a second launch joins the pieces.
// Whole, the CTAs without an item idle for up to steps (1 - items / fit); split, each CTA starts and ends
// two pieces or so. Whole against split, us of GPU time (and of a call from Python, where they differ much),
// heads of 128, groups of 8: 4 items of 3 steps 8.1 and 8.8 (10.9 and 16.1), 7 steps 11.1 and 9.2 (11.7 and
// 16.0); 64 items of 11 steps 14.3 and 18.3, 16 steps 18.3 and 15.9; 256 of 8 steps 19.8 and 28.2; 1024 of 4
// steps 47.5 and 46.7, of uneven 4 steps 39.8 and 62.6. With more columns or dim 256 a step costs more: 16
// items of dim 256, 3 steps 13.7 and 13.3, 4 steps 15.3 and 13.5; 72 of 32 columns, 8 steps 25.0 and 23.0, 16
// steps 37.1 and 31.3. So the rule takes the faster form where there are many items, and the faster call
// where there are few: a captured step loses 2 us there at most, an eager one would lose 5. It misses the
// faster form near its border (64 items of 11 steps are split) and, since items counts what the rows could
// fill at worst, in the last example. At most 16 steps, since one long sequence may be the only one; at most
// four waves of CTAs, since each has to find its item.
struct AttnPlan {
  int64_t ctas, scratch;
  bool whole;
};
template <int D, int NT>
AttnPlan attn_plan(const Dsv41PagedAttnArgs* a) {
  const int64_t group = a->heads / a->kv_heads, slack = 8 * NT - std::gcd<int64_t>(group, 8 * NT);
  const int64_t items = (a->T * group + a->seqs * slack) / (8 * NT) * a->kv_heads;
  int64_t seen = a->width * a->page;
  if (a->window) seen = std::min(seen, a->window + a->T + 15);
  const int64_t steps = cdiv64(cdiv64(seen, 16), PaShape<D, NT>::kWarps);
  const int64_t fit = (int64_t)device_sms() * PaShape<D, NT>::kCtas;
  if (steps <= 16 && items <= 4 * fit && steps * (fit - items) <= (PaShape<D, NT>::kO <= 32 ? 8 : 4) * fit)
    return {std::max<int64_t>(1, items), 0, true};
  const int64_t ctas = std::min(fit, std::max<int64_t>(1, items * steps));
  return {ctas, ctas * (int64_t)(2 * 8 * NT * (D * sizeof(float) + sizeof(float4)) + sizeof(PaSplit)), false};
}

template <int F16, int D, int NT>
int attn_run(const Dsv41PagedAttnArgs* a, void* stream) {
  const AttnPlan plan = attn_plan<D, NT>(a);
  if (plan.scratch && (!a->scratch || a->scratch % 16 || a->scratch_bytes < plan.scratch)) return DSV41_ESCRATCH;
  const uint32_t bits = (uint32_t)a->scale_f32;
  float scale;
  memcpy(&scale, &bits, 4);
  const int64_t slots = 2 * plan.ctas * 8 * NT;
  float* part = ptr<float>(a->scratch);
  const PagedAttnArgs p = {step_rows(a), kv_cache(a), (int)a->heads, (int)a->window, plan.whole, scale * 1.44269504f,
                           ptr<const void>(a->q), ptr<void>(a->out), a->q_ld, a->out_ld, ptr<const float>(a->sink),
                           part, reinterpret_cast<float4*>(part + slots * D),
                           reinterpret_cast<PaSplit*>(part + slots * (D + 4))};
  const dim3 grid((unsigned)plan.ctas);
  const int rc = launch(paged_attn_kernel<F16, D, NT>, grid, dim3(32 * PaShape<D, NT>::kWarps), PaShape<D, NT>::kBytes,
                        stream, p);
  if (rc || plan.whole) return rc;
  return launch(paged_join_kernel<F16, D, NT>, dim3(grid.x, 8 * NT), dim3(kPaJoinThreads), 0, stream, p);
}

}  // namespace

extern "C" {

int dsv41_kv_append(const Dsv41KvAppendArgs* a, void* stream) {
  if (!append_ok(a)) return DSV41_EINVAL;
  if (!a->T || !a->seqs) return DSV41_OK;
  KvAppendArgs k = {step_rows(a), kv_cache(a), (int)a->heads, (int)a->rope,
                    ptr<const void>(a->q), ptr<const void>(a->k), ptr<const void>(a->v), ptr<void>(a->q_out),
                    a->q_ld, a->q_out_ld, a->k_ld, a->v_ld, ptr<const float>(a->cos_sin), a->rope_rows};
  // A warp looks through one row where most rows begin a block of their own (decode and verify rows),
  // else through 16, so that a prompt's warps nearly all find one block. A thread takes one query head
  // while the rows are too few to fill the GPU, else four, for which it reads the angles once.
  k.window = a->T >= 8 * a->seqs ? 16 : 1;
  k.head_step = a->T * a->heads * a->dim / 16 < (int64_t)device_sms() * 2048 ? 1 : 4;
  const int64_t warps = cdiv64(a->T, k.window) * 2 * a->kv_heads;
  const int64_t q_threads = a->q ? a->T * cdiv64(a->heads, k.head_step) * (a->dim / 16) : 0;
  const int64_t kv_ctas = cdiv64(warps, kApThreads / 32), ctas = kv_ctas + cdiv64(q_threads, kApThreads);
  if (ctas > UINT32_MAX / kApThreads) return DSV41_EINVAL;  // threads are counted in 32 bits
  k.kv_ctas = (int)kv_ctas;
  const dim3 grid((unsigned)ctas), cta(kApThreads);
  auto by_pairs = [&](auto f16, auto d) {
    return a->neox ? launch(kv_append_kernel<f16, d, true>, grid, cta, 0, stream, k)
                   : launch(kv_append_kernel<f16, d, false>, grid, cta, 0, stream, k);
  };
  auto by_dim = [&](auto f16) {
    return a->dim == 64 ? by_pairs(f16, Int<64>()) : a->dim == 128 ? by_pairs(f16, Int<128>()) : by_pairs(f16, Int<256>());
  };
  return a->f16 ? by_dim(Int<1>()) : by_dim(Int<0>());
}

int64_t dsv41_paged_attn_scratch_bytes(const Dsv41PagedAttnArgs* a) {
  if (!attn_ok(a)) return DSV41_EINVAL;
  return attn_go(a, [&](auto, auto d, auto nt) { return attn_plan<d, nt>(a).scratch; });
}

int dsv41_paged_attn(const Dsv41PagedAttnArgs* a, void* stream) {
  if (!attn_ok(a)) return DSV41_EINVAL;
  if (!a->T || !a->seqs) return DSV41_OK;
  return (int)attn_go(a, [&](auto f16, auto d, auto nt) { return (int64_t)attn_run<f16, d, nt>(a, stream); });
}

}  // extern "C"
