// The 4-bit products on the 5th-generation tensor cores, for the matrices and row counts where
// reading the weights is what counts (dsv41_gemv_w4; the mma.sync kernel takes the small ones).
//
// 256 weight rows at a time are the M of two accumulators, a thread a row: a converter thread turns
// its row's nibbles into exact bf16 / f16 integers (minus the zero point) and stores them into TMEM as
// the MMA's A operand -- TMEM lane = weight row, so no value crosses threads and nothing is staged in
// shared memory twice; B = the rows of x (N = 16, 32 or 48), staged with the 128-byte swizzle in the
// pair order that the nibble masks give. Every group (or 128 k) has an accumulator of its own, which
// the thread that owns the row reads back and adds to its fp32 sums times the row's scale: scales are
// never rounded into the weights.
//
// 16 warps, one CTA an SM: 0 weight copies (TMA, 256 rows x 128 bytes = 256 k a stage), 1 and 6 the MMA
// issue of the two accumulators, 2 .. 5 x, 8 .. 15 converters. The blocks of all row tiles are cut into equal
// contiguous shares, one a CTA; tiles that lie in several shares are joined from scratch in order by
// a second kernel.
//
// 48 rows of 129280 x 4096, groups of 64: 142 us, 2.1 TB/s of the weights and scales that bound it in
// principle (46 us). The hand-over bounds it now: two converter warps a scheduler each convert, wait for the
// MMA and read back in turn (logic pipe 44 %, tensor pipe 18 %, DRAM 26 %). Weights, x and their
// products are exact; the fp32 sums and y are rounded.
#pragma once

#include "gemv_w4.cuh"
#include "tc_prims.cuh"

namespace dsv41 {

// The nibble mask and the mantissa of 128 (f16: 1024) in registers of their own: as immediates they
// would take two logic instructions a pair instead of one.
template <bool F16>
struct W4Consts {
  uint32_t mask, one;
  __device__ W4Consts() {
    asm volatile("mov.u32 %0, 0x000f000f;" : "=r"(mask));
    asm volatile("mov.u32 %0, %1;" : "=r"(one) : "n"(F16 ? 0x64006400 : 0x43004300));
  }
};
// 8 weights of a word as four pairs (k0, k4), (k1, k5), (k2, k6), (k3, k7) minus their zero point; zz:
// the pair 128 + z (f16: 1024 + z).
template <bool F16>
__device__ __forceinline__ void w4_unpack_z(const W4Consts<F16>& k, uint32_t v, uint32_t zz, uint32_t (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t u;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(u) : "r"(v >> (4 * i)), "r"(k.mask), "r"(k.one));  // (a & b) | c
    if (F16) asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(u), "r"(zz));
    else asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(u), "r"(zz));
  }
}

struct GemvW4TcArgs {
  GemvW4Args a;
  int tiles, kblocks;  // of 256 rows, of 256 k
  float* part;         // [2 CTAs][NP][256] unfinished sums
};

constexpr int kWtThreads = 512;
constexpr int kWtRows = 256;
constexpr int kWtBlock = 256;    // k a stage
constexpr int kWtStages = 4;     // weight stages, 32 KB each
constexpr int kWtXStages = 3;

template <int NP, int SUB>
struct WtShape {
  // accumulators of a unit: as many groups as 128 k hold and 96 columns take; two units' of them where
  // they fit beside two units of A in a half's 256 columns, else one unit's (48 rows of x and groups of
  // 32 or 64)
  static constexpr int kFit = NP == 16 ? 4 : 2;
  static constexpr int kNsub = 128 / SUB < kFit ? 128 / SUB : kFit;
  static constexpr int kDBuf = kNsub * NP <= 64 ? 2 : 1;
  static constexpr int kUnit = SUB * kNsub;  // k between two hand-overs to the tensor core
  static constexpr int kUnits = kWtBlock / kUnit;
  static constexpr int kEntries = kWtBlock / SUB;  // scales a row of a block
  static constexpr int kXStage = NP * kWtBlock * 2;
  static constexpr int kX = kWtStages * kWtRows * 128;
  static constexpr int kBar = kX + kWtXStages * kXStage;
  static constexpr int kNumBars = 2 * kWtStages + 2 * kWtXStages + 12;
  static constexpr int kMisc = kBar + kNumBars * 8;
  static constexpr int kBytes = kMisc + 16 + 1024;
};

// kind::f16, f16 or bf16 inputs, fp32 accumulators, M = 128, N = NP.
template <bool F16>
__device__ __forceinline__ uint32_t wt_idesc(int N) {
  return umma_idesc(128, N, 0, 0) | (F16 ? 0u : (1u << 7) | (1u << 10));
}
// D += A B with A in TMEM.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(db), "r"(idesc), "r"(acc), "r"(0), "r"(0), "r"(0), "r"(0));
}

// Bounded wait that parks the thread (a suspend-time hint), so that the waiting roles leave the issue
// slots to the converters; gives up after 2 s.
__device__ __forceinline__ bool wt_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P1;\n\tmbarrier.try_wait.parity.shared::cta.b64 P1, [%1], %2, %3;\n\t"
      "selp.b32 %0, 1, 0, P1;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(20000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ uint64_t wt_now() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool wt_wait(uint32_t bar, uint32_t parity, volatile int* abort) {
  if (wt_try(bar, parity)) return true;
  const uint64_t deadline = wt_now() + 2000000000ull;
  for (;;) {
    if (wt_try(bar, parity)) return true;
    if (*abort) return false;
    if (wt_now() > deadline) break;
  }
  *abort = 1;
  atomicExch(&g_tc_error, 1);
  return false;
}
// Wait for what is in flight into this CTA's memory, after an abort too (bounded like the others).
__device__ __forceinline__ void wt_land(uint32_t bar, uint32_t parity) {
  const uint64_t deadline = wt_now() + 2000000000ull;
  while (!wt_try(bar, parity) && wt_now() < deadline) {
  }
}

template <bool F16, int NP, int SUB>
__global__ void __launch_bounds__(kWtThreads, 1)
    gemv_w4_tc_kernel(const __grid_constant__ CUtensorMap wmap, const GemvW4TcArgs p) {
  using L = WtShape<NP, SUB>;
  using T = typename Act<F16>::T;
  constexpr int SW = kWtStages, SX = kWtXStages, UK = L::kUnit, NS = L::kNsub, EN = L::kEntries;
  extern __shared__ __align__(1024) uint8_t wt_raw[];
  uint8_t* smem = wt_raw + ((1024 - (smem_u32(wt_raw) & 1023)) & 1023);
  const GemvW4Args& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t bars = smem_u32(smem + L::kBar);
  auto w_full = [&](int s) { return bars + 8 * s; };
  auto w_empty = [&](int s) { return bars + 8 * (SW + s); };
  auto x_full = [&](int s) { return bars + 8 * (2 * SW + s); };
  auto x_empty = [&](int s) { return bars + 8 * (2 * SW + SX + s); };
  auto a_full = [&](int h, int b) { return bars + 8 * (2 * SW + 2 * SX + 2 * h + b); };
  auto d_full = [&](int h, int b) { return bars + 8 * (2 * SW + 2 * SX + 4 + 2 * h + b); };
  auto d_free = [&](int h) { return bars + 8 * (2 * SW + 2 * SX + 10 + h); };  // of the only accumulators
  auto drained = [&](int h) { return bars + 8 * (2 * SW + 2 * SX + 8 + h); };
  uint32_t* tmem_base = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::kMisc + 4);
  if (tid == 0) {
    for (int s = 0; s < SW; ++s) mbar_init(w_full(s), 1), mbar_init(w_empty(s), 8);
    for (int s = 0; s < SX; ++s) mbar_init(x_full(s), 128), mbar_init(x_empty(s), 2);
    for (int h = 0; h < 2; ++h) {
      for (int b = 0; b < 2; ++b) mbar_init(a_full(h, b), 4), mbar_init(d_full(h, b), 1);
      mbar_init(drained(h), 1), mbar_init(d_free(h), 4);
    }
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_base;
  pdl_wait();
  pdl_launch();

  // this CTA's blocks [b0, b1) of all (tile, k block)
  const long long all = (long long)p.tiles * p.kblocks, per = (all + gridDim.x - 1) / gridDim.x;
  const long long b0 = min(blockIdx.x * per, all), b1 = min(b0 + per, all);
  const int blocks = (int)(b1 - b0);
  const int tile0 = (int)(b0 / p.kblocks), kb0 = (int)(b0 % p.kblocks);
  auto units = [&](int kb) { return (min(kWtBlock, a.K - kb * kWtBlock) + UK - 1) / UK; };

  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      for (int tile = tile0, kb = kb0; i < blocks; ++i) {
        const int s = i % SW;
        if (i >= SW && !wt_wait(w_empty(s), ((i / SW) - 1) & 1, abort)) break;
        tc_expect_tx(w_full(s), kWtRows * 128);
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
            "[%4];" ::"r"(smem_u32(smem) + s * kWtRows * 128),
            "l"(&wmap), "r"(kb * 128), "r"(tile * kWtRows), "r"(w_full(s))
            : "memory");
        if (++kb == p.kblocks) kb = 0, ++tile;
      }
      // copies still in flight land before the CTA can exit
      for (int k = max(0, i - SW); k < i; ++k) wt_land(w_full(k % SW), (k / SW) & 1);
    }
  } else if (warp == 1 || warp == 6) {
    if (lane == 0) {
      const int h = warp == 6;
      const uint32_t ta = tmem + 256 * h, td = ta + 128, idesc = wt_idesc<F16>(NP);
      int u = 0;
      bool ok = true;
      for (int i = 0, kb = kb0; ok && i < blocks; ++i) {
        const int xs = i % SX;
        if (!(ok = wt_wait(x_full(xs), (i / SX) & 1, abort))) break;
        const uint32_t sx = smem_u32(smem + L::kX + xs * L::kXStage);
        const int nu = units(kb);
        for (int x = 0; x < nu; ++x, ++u) {
          if (!(ok = wt_wait(a_full(h, u & 1), (u >> 1) & 1, abort))) break;
          if (L::kDBuf == 1 && u && !(ok = wt_wait(d_free(h), (u - 1) & 1, abort))) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < UK / 16; ++k) {
            const int kk = x * UK + 16 * k;  // 64-k chunks of NP rows, 16 k = 32 bytes into a row
            umma_f16_ts(td + (L::kDBuf == 2 ? 64 * (u & 1) : 0) + (16 * k / SUB) * NP, ta + 64 * (u & 1) + 8 * k,
                        umma_sdesc_sw128(sx + (kk >> 6) * NP * 128 + (kk & 63) * 2, 16, 1024), idesc, 16 * k % SUB != 0);
          }
          umma_commit(d_full(h, u & 1));
        }
        if (!ok) break;
        umma_commit(x_empty(xs));
        if (++kb == p.kblocks) kb = 0;
      }
      // and MMAs read and write TMEM before it is freed
      umma_commit(drained(h));
      wt_land(drained(h), 0);
    }
  } else if (warp >= 2 && warp < 6) {
    const int et = tid - 64;
    for (int i = 0, kb = kb0; i < blocks; ++i) {
      const int xs = i % SX;
      if (i >= SX && !wt_wait(x_empty(xs), ((i / SX) - 1) & 1, abort)) break;
      uint8_t* dst = smem + L::kX + xs * L::kXStage;
      uint4 v[NP / 4];
#pragma unroll
      for (int n = 0; n < NP / 4; ++n) {
        const int m = (et >> 5) + 4 * n, k = kb * kWtBlock + 8 * lane;
        v[n] = make_uint4(0, 0, 0, 0);
        if (m < a.M && k < a.K) v[n] = ldg16(reinterpret_cast<const T*>(a.x) + m * a.x_ld + k);
      }
#pragma unroll
      for (int n = 0; n < NP / 4; ++n) {
        const int m = (et >> 5) + 4 * n;
        *reinterpret_cast<uint4*>(dst + (lane >> 3) * NP * 128 + (m >> 3) * 1024 + (m & 7) * 128 +
                                  (((lane & 7) ^ (m & 7)) << 4)) = w4_pair<true>(v[n]);
      }
      fence_async_smem();
      mbar_arrive(x_full(xs));
      if (++kb == p.kblocks) kb = 0;
    }
  } else if (warp >= 8) {
    const int h = (warp - 8) >> 2, row = 128 * h + 32 * (warp & 3) + lane;
    const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ta = tmem + 256 * h + lane_base, td = ta + 128;
    const uint32_t wrow = smem_u32(smem) + row * 128;
    const int groups = a.K / a.group;
    const W4Consts<F16> consts;
    // the scales and zeros of this thread's row in a block, packed; loaded a block ahead
    uint32_t sc[EN / 2], ze[EN > 4 ? 2 : 1], sc_n[EN / 2], ze_n[EN > 4 ? 2 : 1];
    auto load_sz = [&](int tile, int kb) {
      const int64_t r = (int64_t)min(tile * kWtRows + row, a.N - 1) * groups;
      const uint16_t* sp = reinterpret_cast<const uint16_t*>(a.scales) + r;
      if (a.vec) {
        const int64_t at = kb * EN;
        if (EN == 8) {
          const uint4 x = ldg16(sp + at);
          sc_n[0] = x.x, sc_n[1 % (EN / 2)] = x.y, sc_n[2 % (EN / 2)] = x.z, sc_n[3 % (EN / 2)] = x.w;
        } else if (EN == 4) {
          const uint2 x = __ldg(reinterpret_cast<const uint2*>(sp + at));
          sc_n[0] = x.x, sc_n[1 % (EN / 2)] = x.y;
        } else {
          sc_n[0] = __ldg(reinterpret_cast<const uint32_t*>(sp + at));
        }
        if (!a.zeros) {
#pragma unroll
          for (auto& z : ze_n) z = 0x08080808u;
        } else if (EN == 8) {
          const uint2 x = __ldg(reinterpret_cast<const uint2*>(a.zeros + r + at));
          ze_n[0] = x.x, ze_n[EN > 4] = x.y;
        } else if (EN == 4) {
          ze_n[0] = __ldg(reinterpret_cast<const uint32_t*>(a.zeros + r + at));
        } else {
          ze_n[0] = __ldg(reinterpret_cast<const uint16_t*>(a.zeros + r + at));
        }
        return;
      }
#pragma unroll
      for (auto& z : ze_n) z = 0x08080808u;
#pragma unroll
      for (int e = 0; e < EN; ++e) {
        const int g = min(kb * kWtBlock + e * SUB, a.K - 1) / a.group;
        const uint32_t s = __ldg(sp + g);
        sc_n[e / 2] = e & 1 ? sc_n[e / 2] | s << 16 : s;
        if (a.zeros) {
          const uint32_t z = __ldg(a.zeros + r + g);
          ze_n[e / 4] = e & 3 ? ze_n[e / 4] | z << (8 * (e & 3)) : z;
        }
      }
    };
    float acc[NP];
#pragma unroll
    for (int m = 0; m < NP; ++m) acc[m] = 0.f;
    // the unit whose accumulators are not read yet: its scales, and where its tile's sums go if it is
    // the last of its tile here (0: it is not, 1: y, 2: scratch)
    float held[NS];
    int out = 0, out_tile = 0, out_slot = 0;
    bool pending = false;
    int u = 0;
    auto drain = [&]() -> bool {
      const int v = u - 1;
      if (!__all_sync(0xffffffffu, wt_wait(d_full(h, v & 1), (v >> 1) & 1, abort))) return false;
      tc_fence_after();
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int c = 0; c < NP; c += 16) {
          uint32_t d[16];
          tmem_ld16(td + (L::kDBuf == 2 ? 64 * (v & 1) : 0) + s * NP + c, d);
          tmem_wait_ld();
#pragma unroll
          for (int m = 0; m < 16; ++m) acc[c + m] = fmaf(__uint_as_float(d[m]), held[s], acc[c + m]);
        }
      if (L::kDBuf == 1) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(d_free(h));
      }
      if (out) {
        const int n = out_tile * kWtRows + row;
        if (out == 1) {
          T* y = reinterpret_cast<T*>(a.y) + n;
#pragma unroll
          for (int m = 0; m < NP; ++m)
            if (m < a.M && n < a.N) y[m * a.y_ld] = Act<F16>::r(acc[m]);
        } else {
          float* y = p.part + (int64_t)out_slot * NP * kWtRows + row;
#pragma unroll
          for (int m = 0; m < NP; ++m)
            if (m < a.M) y[m * kWtRows] = acc[m];
        }
#pragma unroll
        for (int m = 0; m < NP; ++m) acc[m] = 0.f;
      }
      return true;
    };
    bool ok = true;
    if (blocks) load_sz(tile0, kb0);
    int seg_kb = kb0;  // the k block where this tile's sums here begin
    for (int i = 0, tile = tile0, kb = kb0; ok && i < blocks; ++i) {
      const int s = i % SW, nu = units(kb);
#pragma unroll
      for (int e = 0; e < EN / 2; ++e) sc[e] = sc_n[e];
#pragma unroll
      for (int e = 0; e < (EN > 4 ? 2 : 1); ++e) ze[e] = ze_n[e];
      const bool tile_end = kb + 1 == p.kblocks;
      if (i + 1 < blocks) load_sz(tile_end ? tile + 1 : tile, tile_end ? 0 : kb + 1);
      if (!(ok = __all_sync(0xffffffffu, wt_wait(w_full(s), (i / SW) & 1, abort)))) break;
#pragma unroll
      for (int x = 0; x < L::kUnits; ++x) {
        if (x >= nu) break;
#pragma unroll
        for (int q = 0; q < UK / 32; ++q) {
          const int c = x * (UK / 32) + q, e = 32 * c / SUB;  // the row's 16-byte unit, its scale
          const uint4 w = lds16(wrow + s * kWtRows * 128 + ((c ^ (row & 7)) << 4));
          const uint32_t z = (ze[e / 4] >> (8 * (e & 3))) & 15u;
          const uint32_t zz = (z | z << 16) + consts.one;
          uint32_t r[16];
          w4_unpack_z<F16>(consts, w.x, zz, *reinterpret_cast<uint32_t(*)[4]>(r));
          w4_unpack_z<F16>(consts, w.y, zz, *reinterpret_cast<uint32_t(*)[4]>(r + 4));
          w4_unpack_z<F16>(consts, w.z, zz, *reinterpret_cast<uint32_t(*)[4]>(r + 8));
          w4_unpack_z<F16>(consts, w.w, zz, *reinterpret_cast<uint32_t(*)[4]>(r + 12));
          tmem_st16(ta + 64 * (u & 1) + 16 * q, r);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(a_full(h, u & 1));
          if (x == nu - 1) mbar_arrive(w_empty(s));
        }
        if (pending && !(ok = drain())) break;
        pending = true;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          const int e = x * NS + j;
          const float2 f = Act<F16>::unpack(sc[e / 2]);
          held[j] = e & 1 ? f.y : f.x;
        }
        const bool end = x == nu - 1 && (tile_end || i + 1 == blocks);
        out = !end ? 0 : tile_end && seg_kb == 0 ? 1 : 2;
        out_tile = tile;
        out_slot = 2 * blockIdx.x + (tile == tile0 ? 0 : 1);
        ++u;
      }
      if (tile_end) kb = 0, seg_kb = 0, ++tile;
      else ++kb;
    }
    if (ok && pending) drain();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// Join the pieces of the tile that begins in share blockIdx.x and goes on past its end (at most one),
// in the order of the shares. Thread = weight row.
template <bool F16, int NP>
__global__ void __launch_bounds__(kWtRows) gemv_w4_join_kernel(const GemvW4TcArgs p) {
  using T = typename Act<F16>::T;
  pdl_wait();
  const GemvW4Args& a = p.a;
  const int c = blockIdx.x;
  const long long all = (long long)p.tiles * p.kblocks, per = (all + gridDim.x - 1) / gridDim.x;
  const long long first = c * per, last = min(first + per, all);
  if (first >= all) return;
  const int tile = (int)((last - 1) / p.kblocks);
  const long long t0 = (long long)tile * p.kblocks, t1 = t0 + p.kblocks;
  if (t0 < first || t1 <= last) return;
  const int pieces = (int)((t1 - 1) / per) - c + 1;
  const int n = tile * kWtRows + threadIdx.x;
  if (n >= a.N) return;
  for (int m = blockIdx.y; m < a.M; m += gridDim.y) {
    float s = 0.f;
#pragma unroll 4
    for (int i = 0; i < pieces; ++i) {
      const int64_t slot = 2 * (c + i) + (i == 0 && t0 != first ? 1 : 0);
      s += p.part[(slot * NP + m) * kWtRows + threadIdx.x];
    }
    reinterpret_cast<T*>(a.y)[m * a.y_ld + n] = Act<F16>::r(s);
  }
}

}  // namespace dsv41
