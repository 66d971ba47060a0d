// Products of a few rows with 4-bit weights under group scales (dsv41_gemv_w4):
// y[m][n] = sum over groups of s[n][g] * sum over k in g of x[m][k] (w[n][k] - z[n][g]).
//
// The weights are the bytes that count (half a byte each), so they are read once, in place, and
// everything else rides along. What bounds the kernel beside them is the logic pipe that takes them
// apart, so a nibble n goes into the tensor core as it stands: alone in the low mantissa bits it is
// the subnormal n 2^-24 of f16 (n 2^-133 of bf16), exact like every product of m16n8k16 with x (bf16 x
// is staged times 2^64, so that products stay in fp32's normal range down to x = 2^-57; smaller ones keep
// an absolute 2^-80). Zero points come off the fp32 sums: sum x (n - z) = sum x n - z sum x, the last sum
// taken once with the rows of x in shared memory (where they do not fit, by the same instruction from a
// fragment of ones). So what the additions lose goes by sum |x| (n + z), not by sum |x (n - z)|: for weights
// spread over 0 .. 15 about four times as much, and a group whose weights all equal its zero point leaves
// that instead of exactly 0. Taking z off before the product costs a fourth of the logic instructions.
// Weight rows are the mma's M, the rows of x its N. One word of a lane holds 8 consecutive k of a row;
// masking word >> 4 i gives the pair (k_i, k_(i + 4)), and x is paired up the same way, so no nibble is
// moved for order's sake: 7 logic instructions for 8 weights.
//
// A CTA takes 16 R weight rows at a time, its warps chunks of 256 k (128 bytes a row) in turn; every
// warp streams its chunks through a ring of its own by 16-byte cp.async, across row tiles without a
// pause. The warps' sums meet in shared memory in warp order, so the result does not depend on timing.
//
// One row: 1024 x 1024 2.3 us (launch and one latency), 8192 x 4096 6.5 us (2.7 TB/s: a tile a CTA and two
// chunks a warp, of which the second waits until x is staged),
// 65536 x 8192 at 4.3 TB/s, where the logic pipe issues 63 % of what it can and DRAM is at 53 %.
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
  int gdiv;  // scale entries a group (1: an entry is a group)
};

// NT: tiles of 8 rows of x. R: tiles of 16 weight rows. GS: 32-k steps that share a scale, as far as
// a chunk can know: the largest of 8, 4, 2, 1 with 32 GS dividing the group.
template <int NT, int R, int GS, bool ST>
struct W4Shape {
  static constexpr int kRows = 16 * R;
  static constexpr int kEntries = 8 / GS;                     // scales a row of a chunk
  // weights; without a table of the tile's scales {-zero, scale} of each entry and row
  static constexpr int kStage = kRows * (128 + (ST ? 0 : 8 * kEntries));
  // two or three CTAs an SM beat a deeper ring (N 129280, K 4096, one row: 69 us with 2 stages of 32
  // rows, 92 us with 3 stages and so one CTA)
  static constexpr int kStages = 2;
  static constexpr int kRing = kW4Warps * kStages * kStage;
  // one tile's partial sums, two of them behind the ring; then the rows of x, where they fit
  static __host__ __device__ constexpr int sums(int M) { return kW4Warps * kRows * M * 4; }
  // the scales and zeros of a tile's rows as they lie in memory; one more of them than stages
  static __host__ __device__ constexpr int table(int groups) { return ST ? kRows * groups * 3 : 0; }
  static __host__ __device__ constexpr int before_x(int M, int groups) {
    return kRing + 2 * sums(M) + (kStages + 1) * table(groups);
  }
};

// 8 weights of a word as four pairs (k0, k4), (k1, k5), (k2, k6), (k3, k7) of subnormals.
__device__ __forceinline__ void w4_unpack(uint32_t v, uint32_t (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = (v >> (4 * i)) & 0x000f000fu;
}
// x's 8 values of a word's k in the same pairs; bf16 times 2^64.
template <bool F16>
__device__ __forceinline__ uint4 w4_pair(uint4 x) {
  if (!F16) {
    uint32_t* v[4] = {&x.x, &x.y, &x.z, &x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(*v[i]) : "r"(0x5f805f80u));
  }
  return make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410),
                    __byte_perm(x.y, x.w, 0x7632));
}
// n = 1 as the tensor core sees it: 2^-24 for f16, 2^-133 for bf16.
template <bool F16>
__device__ __forceinline__ float w4_scale() {
  return F16 ? 0x1p-24f : 0x1p-133f;
}
// What turns the fp32 sums into the product's: 2^24 for f16, half of it in the groups' scales and the
// rest on the finished sum, where neither leaves fp32's range; 2^(133 - 64) for bf16, on every group's
// sum, since its scales may take all of fp32's range: an exact multiplication for 32 GS products (one row,
// 27807 x 5728 in groups of 32: 34.2 us for 32.9 without; groups of 64 and more the same with and without).
template <bool F16>
__device__ __forceinline__ float w4_unscale_sum(float sum) {
  return F16 ? sum : sum * 0x1p69f;
}
template <bool F16>
__device__ __forceinline__ float w4_unscale_half() {
  return F16 ? 0x1p12f : 1.f;
}

// 16 bytes at src + o into shared memory, zeros from src + end on.
__device__ __forceinline__ void cp_async16_part(uint32_t dst, const uint8_t* src, int o, int end) {
  const int n = min(max(end - o, 0), 16);
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src + (n ? o : 0)), "r"(n) : "memory");
}

template <bool F16>
__device__ __forceinline__ void w4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  if (F16) mma_f16(c, a0, a1, a2, a3, b0, b1);
  else mma_bf16(c, a0, a1, a2, a3, b0, b1);
}

// XS: x lies in shared memory, paired up once. ST: so do the scales and zeros of whole row tiles, copied
// as they lie a tile ahead; else a warp loads those of each of its chunks.
template <bool F16, int NT, int R, int GS, bool XS, bool ST>
__global__ void __launch_bounds__(32 * kW4Warps) gemv_w4_kernel(const GemvW4Args a) {
  using P = W4Shape<NT, R, GS, ST>;
  using T = typename Act<F16>::T;
  constexpr int W = kW4Warps, S = P::kStages, ROWS = P::kRows, EN = P::kEntries;
  constexpr uint32_t kOnes = 0x00010001u;  // n = 1
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

  // The table of the it-th tile: scales [ROWS][groups], then zeros. The copies for tile it + 1 go out with
  // the first chunk of tile it, so every warp has waited for its share before the barrier that ends tile it.
  uint8_t* tab_p = w4_smem + P::kRing + 2 * P::sums(a.M);
  const int tab_bytes = P::table(groups);
  const int sharers = 32 * min(W, chunks);  // threads of the warps that have chunks
  auto copy_table = [&](int it, int n0) {
    const uint32_t dst = smem_u32(tab_p + it % (S + 1) * tab_bytes);
    const int rows = min(ROWS, a.N - n0), sb = ROWS * groups * 2, zb = sb / 2;
    const uint8_t* sp = reinterpret_cast<const uint8_t*>(a.scales) + (int64_t)n0 * groups * 2;
    const uint8_t* zp = a.zeros + (int64_t)n0 * groups;
    for (int o = tid * 16; o < sb; o += sharers * 16) cp_async16_part(dst + o, sp, o, rows * groups * 2);
    if (a.zeros)
      for (int o = tid * 16; o < zb; o += sharers * 16) cp_async16_part(dst + sb + o, zp, o, rows * groups);
  };

  // Without it a chunk's scales and zeros go through registers: loaded when the chunk is issued, stored (in
  // fp32) when the next one is, so that nothing waits for them.
  uint32_t sc[R][EL], ze[R][EL];
  // the next chunk to issue: its number, its place in the warp's chunks of a tile, the tile
  int is_j = 0, is_c = 0, is_tile = blockIdx.x, is_st = 0, is_it = 0;
  auto load_sz = [&](int k0) {
    const int e0 = EN > 1 ? (lane >> 4) * EL : 0;
    const uint16_t* sp = reinterpret_cast<const uint16_t*>(a.scales);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = (int64_t)min(is_tile * ROWS + 16 * r + (lane & 15), a.N - 1) * groups;
      const int64_t at = row + k0 / (32 * GS) + e0;
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
      } else if (a.vec) {
        sc[r][0] = __ldg(sp + at);
        ze[r][0] = a.zeros ? __ldg(a.zeros + at) : 8;
      } else {
#pragma unroll
        for (int e = 0; e < EL; ++e) {
          const int64_t i = row + min(k0 + 32 * GS * (e0 + e), a.K - 1) / a.group;
          sc[r][e] = __ldg(sp + i);
          ze[r][e] = a.zeros ? __ldg(a.zeros + i) : 8;
        }
      }
    }
  };
  int held = -1;  // the stage they belong to
  auto store_sz = [&] {
    if (held < 0) return;
    uint8_t* p = ring_p + held * P::kStage + ROWS * 128;
    const int e0 = EN > 1 ? (lane >> 4) * EL : 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < EL; ++e) {
        const float z = (float)(ze[r][e] & 15u), s = Act<F16>::unpack(sc[r][e]).x * w4_unscale_half<F16>();
        *reinterpret_cast<float2*>(p + ((e0 + e) * ROWS + 16 * r + (lane & 15)) * 8) = make_float2(-z, s);
      }
    held = -1;
  };
  const int64_t half_k = a.K / 2, row4 = 4 * half_k;
  const uint8_t* w_lane = a.w + (lane / 8) * half_k + warp * (kW4Chunk / 2) + (lane % 8) * 16;
  const uint32_t d_lane = ring + (lane / 8) * 128;  // row's unit c lies at c ^ (row & 7), row & 7 = lane / 8 or that + 4
  auto issue = [&] {
    store_sz();
    if (is_j < total) {
      const int k0 = (warp + is_c * W) * kW4Chunk;
      const uint32_t st = d_lane + is_st * P::kStage;
      const uint8_t* src = w_lane + (int64_t)is_tile * ROWS * half_k + is_c * (W * kW4Chunk / 2);
      if (is_tile * ROWS + ROWS <= a.N && k0 + kW4Chunk <= a.K) {
#pragma unroll
        for (int i = 0; i < 4 * R; ++i, src += row4)
          cp_async16_stream(st + i * 512 + (((lane % 8) ^ (lane / 8 + 4 * (i & 1))) << 4), src);
      } else {
        const bool in = k0 + 32 * (lane % 8) < a.K;
#pragma unroll
        for (int i = 0; i < 4 * R; ++i, src += row4)
          if (in && is_tile * ROWS + lane / 8 + 4 * i < a.N)
            cp_async16_stream(st + i * 512 + (((lane % 8) ^ (lane / 8 + 4 * (i & 1))) << 4), src);
      }
      if (!ST) {
        load_sz(k0);
        held = is_st;
      } else if (is_c == 0 && is_tile + (int)gridDim.x < tiles) {
        copy_table(is_it + 1, (is_tile + gridDim.x) * ROWS);
      }
      ++is_j;
      if (++is_st == S) is_st = 0;
      if (++is_c == mine) is_c = 0, is_tile += gridDim.x, ++is_it;
    }
    cp_async_commit();
  };
  if (ST && tid < sharers) copy_table(0, blockIdx.x * ROWS);
#pragma unroll 1
  for (int i = 0; i < S - 1; ++i) issue();

  // x: rows past M repeat the last one (their columns are never stored)
  uint8_t* x_p = w4_smem + P::before_x(a.M, groups);
  const uint32_t xs = smem_u32(x_p);
  const T* xp[NT];
  uint32_t xa[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int m = min(8 * n + g, a.M - 1);
    xp[n] = reinterpret_cast<const T*>(a.x) + m * a.x_ld + 8 * t;
    xa[n] = xs + (m * 4 + t) * 16;
  }
  // the sums of x over each scale's k, [entry of the row][m] behind the rows of x
  const uint32_t x1 = xs + a.M * a.K * 2;
  if (XS) {
    const int total_x = a.M * (a.K / 8);
    float* sums = reinterpret_cast<float*>(x_p + a.M * a.K * 2);
    for (int i0 = 0; i0 < total_x; i0 += 32 * W) {
      const int i = i0 + tid;
      const bool in = i < total_x;
      const int m = in ? i / (a.K / 8) : 0, c = in ? i % (a.K / 8) : 0;
      float s = 0.f;
      if (in) {
        const uint4 v = w4_pair<F16>(ldg16(reinterpret_cast<const T*>(a.x) + m * a.x_ld + 8 * c));
        *reinterpret_cast<uint4*>(x_p + ((c / 4 * a.M + m) * 4 + c % 4) * 16) = v;
        const uint32_t vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 f = Act<F16>::unpack(vs[q]);
          s += f.x + f.y;
        }
      }
#pragma unroll
      for (int d = 1; d < 4 * GS; d <<= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if (in && c % (4 * GS) == 0) sums[c / (4 * GS) * a.M + m] = s * w4_scale<F16>();
    }
  }
  if (ST) cp_async_wait<S - 2>();  // the first tile's table
  if (XS || ST) __syncthreads();

  float acc[R][NT][4];
  // one staged chunk of `steps` (a full one's 8) 32-k steps, from step k32 of the row on
  auto chunk = [&](uint32_t st, uint32_t tab, int k32, int steps, auto full) {
    // row g's 16-byte unit q lies at unit q ^ g of its 128 bytes
    const uint32_t wq = st + g * 128 + 4 * t + (g << 4), sz = st + ROWS * 128 + g * 8;
    const uint32_t x_step = a.M * 64;
    uint32_t xq[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xq[n] = xa[n] + k32 * x_step;
#pragma unroll
    for (int e = 0; e < EN; ++e) {
      if (!full && e * GS >= steps) break;
      float nz[R][2], sc2[R][2];  // of rows g and g + 8
      uint32_t grp = k32 / GS + e;
      if (ST && a.gdiv > 1) grp /= a.gdiv;
      float d[R][NT][4], d1[NT][4];  // sums of x n, and of x
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        d1[n][0] = d1[n][1] = d1[n][2] = d1[n][3] = 0.f;
        if (XS) {
#pragma unroll
          for (int x = 0; x < 2; ++x)
            asm volatile("ld.shared.f32 %0, [%1];"
                         : "=f"(d1[n][x])
                         : "r"(x1 + (k32 / GS + e) * a.M * 4 + min(8 * n + 2 * t + x, a.M - 1) * 4));
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (ST) {
            const uint32_t at = (16 * r + 8 * h + g) * groups + grp;
            uint32_t v, z = 8;
            asm volatile("ld.shared.u16 %0, [%1];" : "=r"(v) : "r"(tab + 2 * at));
            if (a.zeros) asm volatile("ld.shared.u8 %0, [%1];" : "=r"(z) : "r"(tab + ROWS * groups * 2 + at));
            nz[r][h] = -(float)(z & 15u);
            sc2[r][h] = Act<F16>::unpack(v).x * w4_unscale_half<F16>();
          } else {
            const uint2 v = lds8(sz + (e * ROWS + 16 * r + 8 * h) * 8);
            nz[r][h] = __uint_as_float(v.x);
            sc2[r][h] = __uint_as_float(v.y);
          }
        }
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
            b[n] = w4_pair<F16>(ldg16(xp[n] + 32 * (k32 + q)));
          }
        }
#pragma unroll
        for (int n = 0; n < NT && !XS; ++n) {
          w4_mma<F16>(d1[n], kOnes, kOnes, kOnes, kOnes, b[n].x, b[n].y);
          w4_mma<F16>(d1[n], kOnes, kOnes, kOnes, kOnes, b[n].z, b[n].w);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          uint32_t p[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t v;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"((wq ^ (q << 4)) + (16 * r + 8 * h) * 128));
            w4_unpack(v, p[h]);
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
          for (int x = 0; x < 4; ++x)
            acc[r][n][x] = fmaf(w4_unscale_sum<F16>(fmaf(nz[r][x >> 1], d1[n][x & 1], d[r][n][x])), sc2[r][x >> 1],
                                acc[r][n][x]);
    }
  };
  int rd_st = 0;  // the stage to read
#pragma unroll 1
  for (int i = 0; i < my_tiles; ++i) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[r][n][0] = acc[r][n][1] = acc[r][n][2] = acc[r][n][3] = 0.f;
#pragma unroll 1
    for (int c = 0; c < mine; ++c) {
      const int k0 = (warp + c * W) * kW4Chunk, steps = min(kW4Chunk, a.K - k0) / 32;
      issue();
      cp_async_wait<S - 1>();
      __syncwarp();
      const uint32_t st = ring + rd_st * P::kStage;
      if (++rd_st == S) rd_st = 0;
      const uint32_t tab = smem_u32(tab_p + i % (S + 1) * tab_bytes);
      if (steps == 8) chunk(st, tab, k0 / 32, 8, std::true_type());
      else chunk(st, tab, k0 / 32, steps, std::false_type());
      __syncwarp();
    }
    // the warps' sums, [warp][column][row]
    float* rd = red + (i & 1) * (P::sums(a.M) / 4);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (const int m = 8 * n + 2 * t + (e & 1); m < a.M)
            rd[(warp * a.M + m) * ROWS + 16 * r + g + 8 * (e >> 1)] = acc[r][n][e];
    __syncthreads();
    const int n0 = (blockIdx.x + i * gridDim.x) * ROWS;
    for (int o = tid; o < a.M * ROWS; o += 32 * W) {
      const int m = o / ROWS, row = o % ROWS;
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += rd[(w * a.M + m) * ROWS + row];
      if (n0 + row < a.N) reinterpret_cast<T*>(a.y)[m * a.y_ld + n0 + row] = Act<F16>::r(s * w4_unscale_half<F16>());
    }
  }
}

}  // namespace dsv41
