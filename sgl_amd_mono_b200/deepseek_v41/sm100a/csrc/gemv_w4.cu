// extern "C" entry points of the 4-bit GEMV (include/dsv41_b200.h): argument checks, the choice of the
// kernel, the launches on the caller's stream.
#include <cstdio>

#include "../../../../include/dsv41_b200.h"
#include "gemv_w4.cuh"
#include "gemv_w4_tc.cuh"
#include "gqa_launch.cuh"

using namespace dsv41;

namespace {

// Bytes of its tables of scales and zeros (whole row tiles'); rows of more groups load them chunk by chunk.
constexpr int kW4TableBytes = 32 * 1024;

bool w4_ok(const Dsv41GemvW4Args* a) {
  return a && a->w && a->w % 16 == 0 && a->scales && a->scales % 2 == 0 && a->x && a->x % 16 == 0 && a->y &&
         a->y % 2 == 0 && a->M >= 1 && a->M <= kW4MaxRows && a->N >= 1 && a->N <= (1 << 24) && a->group >= 32 &&
         a->group % 32 == 0 && a->K >= a->group && a->K <= (1 << 24) && a->K % a->group == 0 && a->x_ld % 8 == 0 &&
         a->x_ld >= a->K && a->y_ld >= a->N && (a->f16 == 0 || a->f16 == 1);
}

// Shared memory of a CTA with which two fit an SM.
constexpr int kW4HalfSm = 112 * 1024;

template <int NT, int R, int GS, bool ST>
int w4_go(int64_t f16, GemvW4Args g, void* stream) {
  using P = W4Shape<NT, R, GS, ST>;
  // The rows of x lie in shared memory while two CTAs fit an SM with them; else they are read through
  // L1 (N 129280, K 4096: 3 rows 62 us kept and 70 read, 4 rows 70 either way with one CTA an SM).
  const int64_t x_smem = (int64_t)g.M * g.K * 2 + g.K / (32 * GS) * g.M * 4;
  const int rest = P::before_x(g.M, g.K / g.group);
  const bool xs = NT == 1 && rest + x_smem <= kW4HalfSm;
  const int smem = rest + (xs ? (int)x_smem : 0);
  // persistent: as many CTAs as fit, each taking every grid-th row tile
  const int fit = std::min(std::max(1, 226 * 1024 / (smem + 1024)), 4);
  const dim3 grid(std::min(cdiv(g.N, P::kRows), device_sms() * fit)), block(32 * kW4Warps);
  if constexpr (NT == 1) {
    if (xs)
      return f16 ? launch(gemv_w4_kernel<true, NT, R, GS, true, ST>, grid, block, smem, stream, g)
                 : launch(gemv_w4_kernel<false, NT, R, GS, true, ST>, grid, block, smem, stream, g);
  }
  return f16 ? launch(gemv_w4_kernel<true, NT, R, GS, false, ST>, grid, block, smem, stream, g)
             : launch(gemv_w4_kernel<false, NT, R, GS, false, ST>, grid, block, smem, stream, g);
}

template <int NT, int R, int GS>
int w4_run(int64_t f16, GemvW4Args g, void* stream) {
  using P = W4Shape<NT, R, GS, true>;
  const uintptr_t sp = reinterpret_cast<uintptr_t>(g.scales), zp = reinterpret_cast<uintptr_t>(g.zeros);
  g.gdiv = g.group / (32 * GS);
  if ((P::kStages + 1) * P::table(g.K / g.group) <= kW4TableBytes && sp % 16 == 0 && zp % 16 == 0)
    return w4_go<NT, R, GS, true>(f16, g, stream);
  // a lane's scales of a chunk in one load
  constexpr int el = P::kEntries > 1 ? P::kEntries / 2 : 1;
  g.vec = g.gdiv == 1 && g.K / g.group % el == 0 && g.K % kW4Chunk == 0 && sp % (2 * el) == 0 && zp % el == 0;
  return w4_go<NT, R, GS, false>(f16, g, stream);
}

template <int NT, int R>
int w4_group(int64_t f16, const GemvW4Args& g, void* stream) {
  const int steps = g.group / 32;
  return steps % 8 == 0   ? w4_run<NT, R, 8>(f16, g, stream)
         : steps % 4 == 0 ? w4_run<NT, R, 4>(f16, g, stream)
         : steps % 2 == 0 ? w4_run<NT, R, 2>(f16, g, stream)
                          : w4_run<NT, R, 1>(f16, g, stream);
}

// ------------------------------------------------ the tcgen05 kernel
int w4_tc_rows(const Dsv41GemvW4Args* a) { return a->M <= 16 ? 16 : a->M <= 32 ? 32 : 48; }
// More than 16 rows over a matrix large enough to fill its pipeline (48 rows, K 4096: N 8192 28 us on
// mma.sync and 25 here, N 28672 93 and 45; 4096 x 1024 stays at half the time on mma.sync). From 9 rows
// where mma.sync reads scales often and the matrix is twice that (16 rows, K 4096, mma.sync and here:
// groups of 32 N 8192 17.7 and 19.5, N 28672 57.5 and 37.3; of 64 N 28672 45.9 and 35.6; of 128 32.2 and
// 34.9).
bool w4_tc(const Dsv41GemvW4Args* a) {
  return a->M > 16 ? a->N * a->K >= (32 << 20) : a->M > 8 && a->group % 128 && a->N * a->K >= (64 << 20);
}
int w4_tc_ctas(const Dsv41GemvW4Args* a) {
  return (int)std::min<int64_t>(device_sms(), cdiv64(a->N, kWtRows) * cdiv64(a->K, kWtBlock));
}
int64_t w4_tc_scratch(const Dsv41GemvW4Args* a) {
  return (int64_t)2 * w4_tc_ctas(a) * w4_tc_rows(a) * kWtRows * 4;
}

template <int F16, int NP, int SUB>
int w4_tc_run(const Dsv41GemvW4Args* a, GemvW4Args g, void* stream) {
  using L = WtShape<NP, SUB>;
  g.vec = g.group == SUB && g.K % kWtBlock == 0 && a->scales % (2 * L::kEntries) == 0 && a->zeros % L::kEntries == 0;
  CUtensorMap map;
  if (!byte_tile_map(&map, g.w, g.N, g.K / 2)) {
    fprintf(stderr, "dsv41: 4-bit weight tensor map failed\n");
    return DSV41_ELAUNCH;
  }
  const GemvW4TcArgs t = {g, cdiv(g.N, kWtRows), cdiv(g.K, kWtBlock), ptr<float>(a->scratch)};
  const int ctas = w4_tc_ctas(a);
  const int rc = launch(gemv_w4_tc_kernel<F16, NP, SUB>, dim3(ctas), dim3(kWtThreads), L::kBytes, stream, map, t);
  return rc ? rc : launch(gemv_w4_join_kernel<F16, NP>, dim3(ctas, cdiv(g.M, 8)), dim3(kWtRows), 0, stream, t);
}

template <int NP>
int w4_tc_group(const Dsv41GemvW4Args* a, const GemvW4Args& g, void* stream) {
  const int steps = g.group / 32;
  if (steps % 4 == 0)
    return a->f16 ? w4_tc_run<1, NP, 128>(a, g, stream) : w4_tc_run<0, NP, 128>(a, g, stream);
  if (steps % 2 == 0) return a->f16 ? w4_tc_run<1, NP, 64>(a, g, stream) : w4_tc_run<0, NP, 64>(a, g, stream);
  return a->f16 ? w4_tc_run<1, NP, 32>(a, g, stream) : w4_tc_run<0, NP, 32>(a, g, stream);
}

}  // namespace

bool dsv41::gqa_device_error(int* v) { return cudaMemcpyFromSymbol(v, g_tc_error, sizeof(*v)) == cudaSuccess; }

extern "C" {

int64_t dsv41_gemv_w4_scratch_bytes(const Dsv41GemvW4Args* a) {
  if (!w4_ok(a)) return DSV41_EINVAL;
  return w4_tc(a) ? w4_tc_scratch(a) : 0;
}


int dsv41_gemv_w4(const Dsv41GemvW4Args* a, void* stream) {
  if (!w4_ok(a)) return DSV41_EINVAL;
  GemvW4Args g = {ptr<const uint8_t>(a->w), ptr<const void>(a->scales), ptr<const uint8_t>(a->zeros),
                  ptr<const void>(a->x), ptr<void>(a->y), (int)a->M, (int)a->N, (int)a->K, (int)a->group,
                  a->x_ld, a->y_ld, 0, 1};
  if (w4_tc(a)) {
    if (!a->scratch || a->scratch % 16 || a->scratch_bytes < w4_tc_scratch(a)) return DSV41_ESCRATCH;
    return g.M <= 16   ? w4_tc_group<16>(a, g, stream)
           : g.M <= 32 ? w4_tc_group<32>(a, g, stream)
                       : w4_tc_group<48>(a, g, stream);
  }
  // 32 weight rows a warp share its fragments of x; 16 make more work items of a small matrix (one row,
  // K 4096: N 1024 2.3 us with 16 and 2.5 with 32; N 4096 5.4 and 5.4; N 8192 8.7 and 7.4)
  if (g.M <= 8) return g.N >= 4096 ? w4_group<1, 2>(a->f16, g, stream) : w4_group<1, 1>(a->f16, g, stream);
  return g.M <= 16   ? w4_group<2, 2>(a->f16, g, stream)
         : g.M <= 32 ? w4_group<4, 2>(a->f16, g, stream)
                     : w4_group<6, 2>(a->f16, g, stream);
}

}  // extern "C"
