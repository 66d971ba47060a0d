// Products of a few rows with 4-bit weights under group scales (dsv41_gemv_w4):
// y[m][n] = sum over groups of s[n][g] * sum over k in g of x[m][k] (w[n][k] - z[n][g]).
//
// The weights are the bytes that count (half a byte each), so they are read once, in place, and
// everything else rides along. A weight becomes a bf16 (f16) by placing its nibble in the mantissa of
// 128 (1024) and subtracting 128 + z (1024 + z): both exact, so a product of m16n8k16 is exact in
// fp32 and the group's scale multiplies the fp32 sum of every 32 k. Weight rows are the mma's M, the
// rows of x its N. One word of a lane holds 8 consecutive k of a row; masking word >> 4 i gives the
// pair (k_i, k_(i + 4)), and x is paired up the same way, so no nibble is moved for order's sake.
//
// A CTA takes 16 R weight rows at a time, its warps chunks of 256 k (128 bytes a row) in turn; every
// warp streams its chunks through a ring of its own by 16-byte cp.async, across row tiles without a
// pause. The warps' sums meet in shared memory in warp order, so the result does not depend on timing.
#pragma once

#include <type_traits>

#include "gqa.cuh"

namespace dsv41 {

constexpr int kW4MaxRows = 48;
constexpr int kW4Warps = 8;
constexpr int kW4Chunk = 256;  // k a stage

struct GemvW4Args {
  const uint8_t* w;
  const void* scales;
  const uint8_t* zeros;  // or null: 8
  const void* x;
  void* y;
  int M, N, K, group;
  int64_t x_ld, y_ld;
  int vec;  // a lane's scales of a chunk, and its zeros, can be read in one load each
};

// NT: tiles of 8 rows of x. R: tiles of 16 weight rows. GS: 32-k steps that share a scale, as far as
// a chunk can know: the largest of 8, 4, 2, 1 with 32 GS dividing the group.
template <int NT, int R, int GS>
struct W4Shape {
  static constexpr int kRows = 16 * R;
  static constexpr int kEntries = 8 / GS;                     // scales a row of a chunk
  static constexpr int kStage = kRows * (128 + 8 * kEntries);  // weights; {zero pair, scale} of each entry and row
    // two or three CTAs an SM beat a deeper ring (N 129280, K 4096, one row: 69 us with 2 stages of 32
  // rows, 92 us with 3 stages and so one CTA)
  static constexpr int kStages = R == 1 ? 3 : 2;
  static constexpr int kRed = kW4Warps * kRows * 8 * NT * 4;  // one tile's partial sums
  static constexpr int kRing = kW4Warps * kStages * kStage;
  static constexpr int kBytes = kRing + 2 * kRed;             // and the rows of x, where they fit
};

// The nibble mask and the mantissa of 128 (f16: 1024) in registers of their own: as immediates they
// would take two logic instructions a pair instead of one, on the pipe that bounds the kernel.
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
__device__ __forceinline__ void w4_unpack(const W4Consts<F16>& k, uint32_t v, uint32_t zz, uint32_t (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t u;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(u) : "r"(v >> (4 * i)), "r"(k.mask), "r"(k.one));  // (a & b) | c
    if (F16) asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(u), "r"(zz));
    else asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(u), "r"(zz));
  }
}
// x's 8 values of a word's k in the same pairs.
__device__ __forceinline__ uint4 w4_pair(uint4 x) {
  return make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410),
                    __byte_perm(x.y, x.w, 0x7632));
}

template <bool F16>
__device__ __forceinline__ void w4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  if (F16) mma_f16(c, a0, a1, a2, a3, b0, b1);
  else mma_bf16(c, a0, a1, a2, a3, b0, b1);
}

// XS: x lies in shared memory, paired up once (behind the ring and the sums).
template <bool F16, int NT, int R, int GS, bool XS>
__global__ void __launch_bounds__(32 * kW4Warps) gemv_w4_kernel(const GemvW4Args a) {
  using P = W4Shape<NT, R, GS>;
  using T = typename Act<F16>::T;
  constexpr int W = kW4Warps, S = P::kStages, ROWS = P::kRows, EN = P::kEntries;
  constexpr int EL = EN > 1 ? EN / 2 : 1;  // entries a lane loads: lanes 0 .. 15 the first half, 16 .. 31 the other
  extern __shared__ __align__(128) uint8_t w4_smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  uint8_t* ring_p = w4_smem + warp * S * P::kStage;
  const uint32_t ring = smem_u32(ring_p);
  float* red = reinterpret_cast<float*>(w4_smem + P::kRing);
  const int chunks = (a.K + kW4Chunk - 1) / kW4Chunk, groups = a.K / a.group;
  const int tiles = (a.N + ROWS - 1) / ROWS;
  const int mine = (chunks - warp + W - 1) / W;  // this warp's chunks of a tile
  const int my_tiles = (tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  const int total = mine > 0 ? mine * my_tiles : 0;
  pdl_wait();

  // A chunk's scales and zeros go through registers: loaded when the chunk is issued, stored (as fp32
  // scale and zero pair) when the next one is, so that nothing waits for them.
  uint32_t sc[R][EL], ze[R][EL];
  int held = -1;  // the chunk they belong to
  auto load_sz = [&](int j) {
    const int tile = blockIdx.x + j / mine * gridDim.x, k0 = (warp + j % mine * W) * kW4Chunk;
    const int e0 = EN > 1 ? (lane >> 4) * EL : 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = (int64_t)min(tile * ROWS + 16 * r + (lane & 15), a.N - 1) * groups;
      const int64_t at = row + (k0 + 32 * GS * e0) / a.group;
      const uint16_t* sp = reinterpret_cast<const uint16_t*>(a.scales);
      if (a.vec && EL == 4) {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(sp + at));
        sc[r][0] = x.x & 0xffff, sc[r][1 % EL] = x.x >> 16, sc[r][2 % EL] = x.y & 0xffff, sc[r][3 % EL] = x.y >> 16;
        const uint32_t z = a.zeros ? __ldg(reinterpret_cast<const uint32_t*>(a.zeros + at)) : 0x08080808u;
#pragma unroll
        for (int e = 0; e < EL; ++e) ze[r][e] = z >> (8 * e);
      } else if (a.vec && EL == 2) {
        const uint32_t x = __ldg(reinterpret_cast<const uint32_t*>(sp + at));
        sc[r][0] = x & 0xffff, sc[r][1 % EL] = x >> 16;
        const uint32_t z = a.zeros ? __ldg(reinterpret_cast<const uint16_t*>(a.zeros + at)) : 0x0808u;
        ze[r][0] = z, ze[r][1 % EL] = z >> 8;
      } else {
#pragma unroll
        for (int e = 0; e < EL; ++e) {
          const int64_t i = row + min(k0 + 32 * GS * (e0 + e), a.K - 1) / a.group;
          sc[r][e] = __ldg(sp + i);
          ze[r][e] = a.zeros ? __ldg(a.zeros + i) : 8;
        }
      }
    }
    held = j;
  };
  auto store_sz = [&] {
    if (held < 0) return;
    uint8_t* p = ring_p + held % S * P::kStage + ROWS * 128;
    const int e0 = EN > 1 ? (lane >> 4) * EL : 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < EL; ++e) {
        const uint32_t z = ze[r][e] & 15u;
        const float2 s = Act<F16>::unpack(sc[r][e]);
        *reinterpret_cast<uint2*>(p + ((e0 + e) * ROWS + 16 * r + (lane & 15)) * 8) =
            make_uint2((z | z << 16) + (F16 ? 0x64006400u : 0x43004300u), __float_as_uint(s.x));
      }
    held = -1;
  };
  auto issue = [&](int j) {
    store_sz();
    if (j < total) {
      const int tile = blockIdx.x + j / mine * gridDim.x, k0 = (warp + j % mine * W) * kW4Chunk;
      const uint32_t st = ring + j % S * P::kStage;
      const int bytes = min(kW4Chunk, a.K - k0) / 2;
#pragma unroll
      for (int i = 0; i < 4 * R; ++i) {
        const int row = lane / 8 + 4 * i, c = lane % 8;
        if (c * 16 < bytes)
          cp_async16_stream(st + row * 128 + ((c ^ (row & 7)) << 4),
                            a.w + (int64_t)min(tile * ROWS + row, a.N - 1) * (a.K / 2) + k0 / 2 + c * 16);
      }
      load_sz(j);
    }
    cp_async_commit();
  };
#pragma unroll 1
  for (int j = 0; j < S - 1; ++j) issue(j);

  // x: rows past M repeat the last one (their columns are never stored)
  const uint32_t xs = smem_u32(w4_smem + P::kBytes);
  const T* xp[NT];
  uint32_t xa[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int m = min(8 * n + g, a.M - 1);
    xp[n] = reinterpret_cast<const T*>(a.x) + m * a.x_ld + 8 * t;
    xa[n] = xs + (m * 4 + t) * 16;
  }
  if (XS) {
    for (int i = tid; i < a.M * (a.K / 8); i += 32 * W) {
      const int m = i / (a.K / 8), c = i % (a.K / 8);
      const uint4 v = w4_pair(ldg16(reinterpret_cast<const T*>(a.x) + m * a.x_ld + 8 * c));
      *reinterpret_cast<uint4*>(w4_smem + P::kBytes + ((c / 4 * a.M + m) * 4 + c % 4) * 16) = v;
    }
    __syncthreads();
  }

  const W4Consts<F16> consts;
  float acc[R][NT][4];
  // one staged chunk of `steps` (a full one's 8) 32-k steps, from step k32 of the row on
  auto chunk = [&](uint32_t st, int k32, int steps, auto full) {
    // row g's 16-byte unit q lies at unit q ^ g of its 128 bytes
    const uint32_t wq = st + g * 128 + 4 * t + (g << 4), sz = st + ROWS * 128 + g * 8;
    const uint32_t x_step = a.M * 64;
    uint32_t xq[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xq[n] = xa[n] + k32 * x_step;
#pragma unroll
    for (int e = 0; e < EN; ++e) {
      if (!full && e * GS >= steps) break;
      uint2 zs[R][2];  // rows g and g + 8
      float d[R][NT][4];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        zs[r][0] = lds8(sz + (e * ROWS + 16 * r) * 8);
        zs[r][1] = lds8(sz + (e * ROWS + 16 * r + 8) * 8);
#pragma unroll
        for (int n = 0; n < NT; ++n) d[r][n][0] = d[r][n][1] = d[r][n][2] = d[r][n][3] = 0.f;
      }
#pragma unroll
      for (int u = 0; u < GS; ++u) {
        const int q = e * GS + u;
        if (!full && GS > 1 && q >= steps) break;
        uint4 b[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (XS) {
            b[n] = lds16(xq[n]);
            xq[n] += x_step;
          } else {
            b[n] = w4_pair(ldg16(xp[n] + 32 * (k32 + q)));
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          uint32_t p[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t v;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"((wq ^ (q << 4)) + (16 * r + 8 * h) * 128));
            w4_unpack<F16>(consts, v, zs[r][h].x, p[h]);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            w4_mma<F16>(d[r][n], p[0][0], p[1][0], p[0][1], p[1][1], b[n].x, b[n].y);
            w4_mma<F16>(d[r][n], p[0][2], p[1][2], p[0][3], p[1][3], b[n].z, b[n].w);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[r][n][x] = fmaf(d[r][n][x], __uint_as_float(zs[r][x >> 1].y), acc[r][n][x]);
    }
  };
  int j = 0;
#pragma unroll 1
  for (int i = 0; i < my_tiles; ++i) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[r][n][0] = acc[r][n][1] = acc[r][n][2] = acc[r][n][3] = 0.f;
#pragma unroll 1
    for (int c = 0; c < mine; ++c, ++j) {
      const int k0 = (warp + c * W) * kW4Chunk, steps = min(kW4Chunk, a.K - k0) / 32;
      issue(j + S - 1);
      cp_async_wait<S - 1>();
      __syncwarp();
      const uint32_t st = ring + j % S * P::kStage;
      if (steps == 8) chunk(st, k0 / 32, 8, std::true_type());
      else chunk(st, k0 / 32, steps, std::false_type());
      __syncwarp();
    }
    // the warps' sums, [warp][column][row]
    float* rd = red + (i & 1) * (P::kRed / 4);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          rd[(warp * 8 * NT + 8 * n + 2 * t + (e & 1)) * ROWS + 16 * r + g + 8 * (e >> 1)] = acc[r][n][e];
    __syncthreads();
    const int n0 = (blockIdx.x + i * gridDim.x) * ROWS;
    for (int o = tid; o < a.M * ROWS; o += 32 * W) {
      const int m = o / ROWS, row = o % ROWS;
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += rd[(w * 8 * NT + m) * ROWS + row];
      if (n0 + row < a.N) reinterpret_cast<T*>(a.y)[m * a.y_ld + n0 + row] = Act<F16>::r(s);
    }
  }
}

}  // namespace dsv41
