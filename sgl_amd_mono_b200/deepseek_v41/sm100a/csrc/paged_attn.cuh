// Attention of decode and verify rows over the paged e4m3 cache (dsv41_paged_attn).
//
// Mathematics. For a row's query head with scores s_i = scale q . k_i (base 2: scale log2 e), keys
// k_i = 2^a_i K_i and values v_i = 2^b_i V_i (K, V e4m3 bytes, a and b one power of two per block
// of tokens and head): o = 2^(r - c) sum_i 2^(s_i + b_i - r) V_i / sum_i 2^(s_i - c), one pass with
// two running references. The value's scale goes into the weight's exponent, so the weights w_i =
// 2^(s_i + b_i - r + 7) multiply raw bytes; r follows the largest s_i + b_i seen, c the largest s_i
// (two, since a scale may be any power of two: one reference could overflow the sum). Both move only
// when a weight would pass 2^15 (or a term of the sum 2^60), so most tiles rescale nothing.
//
// Layout. What bounds the kernel is reading the cache once, so all columns (a sequence's rows times
// the query heads of a kv head) that fit share each tile. A tile is 16 tokens of one kv head: 16 dim
// contiguous bytes of K and of V, never across a page or a scale block. A warp streams its own tiles
// through its own ring of shared memory by 16-byte cp.async, with no barrier between warps; S^T = K
// Q^T puts the 16 tokens in the m16n8k16 rows and 8 columns in N, so a group of 8 heads or fewer
// wastes little, and O^T = V^T P^T takes P from S's registers by a transposing movmatrix.
//
// Roundings. K and V become f16 exactly; q is scaled per column by a power of two into f16's range
// (exact but for values 2^-29 below the column's largest). Scores, weights, sums and O are fp32. A
// weight enters the second product as two f16 numbers, its head and what the head leaves, which
// keeps it to 2^-22 of itself and 2^-32 of the column's largest. The head alone (2^-11) showed: outputs
// 8e-4 (bf16) and 3e-4 (f16) of their size away from those of fp32 weights, now 1e-4 or less (bf16, 131072
// tokens: up to 1.7e-4). The tails' product costs 2 % with one column tile (95 to 97 us for 48 rows at 8192
// tokens, 182 to 186 for 4 at 131072) and 13 % with three (147 to 167). What is left over long contexts is
// the tensor core's truncation of its fp32 sums, up to 2^-23 of O a product: each tile's product by
// itself and added to O with rounding has 2e-5 at 131072 tokens, but costs 9 to 11 % (spills; 108 us, 203
// and 183), and is left out.
//
// Split. The work (sequence, kv head, column tile, steps of 16 W tokens) is cut into equal
// contiguous shares, one a CTA, whatever the lengths: each CTA finds its own from the lengths on the
// device. A share's piece of an item that lies in several shares goes to scratch, and a second kernel
// joins the pieces in order, so the sums do not depend on timing. Where pages or window keep
// the items short, and there are not a few items only, they are not split and one launch does.
//
// 4 rows of 64 heads over 131072 tokens, 8 kv heads: 186 us, its bytes take 0.88 of that. With up to 16
// columns DRAM bounds it; with more, latencies between the dependent products and conversions of a tile
// on the two or three warps a scheduler that their registers leave (8 x 6 rows, 24 columns, at 32768
// tokens: 167 us for 82 us of bytes), some of which spill (24 columns of 128 dims: 255 registers, 232
// bytes reloaded in bf16 and 208 in f16).
#pragma once

#include <cfloat>

#include "gqa.cuh"

namespace dsv41 {

struct PagedAttnArgs {
  StepRows rows;
  KvCache cache;
  int heads, window;
  int whole;    // items are not split: a CTA each, no scratch and no second kernel
  float scale;  // times log2 e
  const void* q;
  void* out;
  int64_t q_ld, out_ld;
  const float* sink;  // [heads] or null
  float* part;        // [2 CTAs][8 NT][dim] unnormalised pieces
  float4* part_rl;    // [2 CTAs][8 NT] their references r and c and their sum
  struct PaSplit* split;  // [CTAs]
};

// The item that begins in a share and goes on in the next ones, if one does: its pieces (0: none), what
// its columns are, and the slot of its first piece (the others lie in the slots 2 (share + i)).
struct PaSplit {
  int pieces, slot, row0, h0, col0, cols, pad[2];
};

// One sequence's work: its rows, its tiles [tile0, tile0 + tiles) and what that makes in units.
struct SeqWork {
  int row0, n, cols, cts, tile0, tiles, steps, end;  // end: tokens its last row sees, up to 2^31 - 1
  long long units;
};

// The first token that a row sees which sees the tokens before vis. (A row before the sequence's first
// token has vis <= 0, and a window may be 2^31 - 1, so their difference need not fit 32 bits.)
__device__ __forceinline__ int window_low(int vis, int window) { return window && vis > window ? vis - window : 0; }

template <int NT, int W>
__device__ __forceinline__ SeqWork seq_work(const PagedAttnArgs& a, int s) {
  SeqWork w;
  w.row0 = a.rows.cu_rows ? a.rows.cu_rows[s] : s;
  w.n = a.rows.cu_rows ? a.rows.cu_rows[s + 1] - w.row0 : 1;
  w.n = w.row0 < 0 || w.row0 > a.rows.T ? 0 : max(0, min(w.n, a.rows.T - w.row0));
  w.end = max(a.rows.lens[s], 0);
  const int kvh = a.cache.kv_heads;
  w.cols = w.n * (a.heads / kvh);
  w.cts = (w.cols + 8 * NT - 1) / (8 * NT);
  const int hi = min(w.end, a.rows.width * a.cache.page);
  w.tile0 = window_low(w.end - w.n + 1, a.window) / 16;
  w.tiles = max(0, (hi + 15) / 16 - w.tile0);
  w.steps = max(1, (w.tiles + W - 1) / W);
  w.units = (long long)w.cts * kvh * (a.whole ? 1 : w.steps);
  return w;
}

// The whole work and this share of it: seq and unit where share `c` of `shares` begins, found by all
// threads of a CTA of W warps. per = units a share.
struct Share {
  long long first, last, per;  // units [first, last)
  int seq;                     // the sequence of unit `first`
  long long seq0;              // its first unit
};

template <int NT, int W>
__device__ __forceinline__ Share find_share(const PagedAttnArgs& a, int c, int shares, long long* sm) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kThreads = 32 * W;
  const int seqs = a.rows.seqs;
  // the units before each thread's sequence, a chunk of kThreads sequences at a time
  auto scan = [&](int base, long long& before, long long& own) {
    own = base + tid < seqs ? seq_work<NT, W>(a, base + tid).units : 0;
    long long x = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 31) sm[warp] = x;
    __syncthreads();
    before = x - own;
    long long all = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (i < warp) before += sm[i];
      all += sm[i];
    }
    return all;
  };
  long long before, own, total = scan(0, before, own);
  for (int base = kThreads; base < seqs; base += kThreads) {
    long long b, o;
    total += scan(base, b, o);
  }
  Share r;
  r.per = (total + shares - 1) / shares;
  r.first = c * r.per;
  r.last = min(r.first + r.per, total);
  if (r.first >= total) return r.seq = -1, r;
  __syncthreads();
  long long sum = 0;
  for (int base = 0; base < seqs; base += kThreads) {
    if (seqs > kThreads) {
      const long long all = scan(base, before, own);
      before += sum;
      sum += all;
    }
    if (own && before <= r.first && r.first < before + own) {
      sm[W] = base + tid;
      sm[W + 1] = before;
    }
  }
  __syncthreads();
  r.seq = (int)sm[W];
  r.seq0 = sm[W + 1];
  return r;
}

// A tile's token rows in the mma's M order: row g is token kappa(g) (g + 8: 8 more). With the
// swizzle below every shared-memory read of K and V is free of bank conflicts.
__device__ __forceinline__ int pa_kappa(int g) { return (g & 1) ? 7 - (g >> 1) : g >> 1; }
// Where 16-byte chunk c of token row `row` lies in a staged tile.
template <int D>
__device__ __forceinline__ uint32_t pa_chunk(int row, int c) {
  return row * D + ((D == 64 ? c ^ (row & 2) : c ^ (row & 7)) << 4);
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// f16x2 of the low and of the high two e4m3 bytes of w (exact, NaN kept).
__device__ __forceinline__ void e4m3x4_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h; }"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
// m16n8k16 of f16 and a shared-memory load that the compiler may schedule freely.
__device__ __forceinline__ void pa_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <class V>
__device__ __forceinline__ V pa_lds(const uint8_t* p) {
  return *reinterpret_cast<const V*>(p);
}
// The bytes of w that are e4m3 NaN, as a mask.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }

template <int D, int NT>
struct PaShape {
  // What a thread holds decides how many warps an SM runs: two CTAs of 8 while O takes up to 32 registers
  // (and the fragments of Q as many), one of 12 up to 64, else one of 8 (8 sequences at 32768 tokens, dim
  // 128: O of 64 123 us with 12 warps, 128 with two CTAs of 8, 126 with 8; O of 96 179 us with 12 and 171 with 8;
  // dim 256 at 16384 tokens, O of 64: 104, 108 and 99).
  static constexpr int kO = NT * D / 4;               // O registers a thread
  static constexpr int kCtas = kO <= 32 ? 2 : 1;      // an SM
  static constexpr int kWarps = kO <= 32 || kO > 64 ? 8 : 12;
  static constexpr int kTile = 32 * D;                // bytes of a staged tile, K and V
  static constexpr int kStagesFit = 192 / kCtas * 1024 / (kWarps * kTile);
  static constexpr int kStages = kStagesFit > 6 ? 6 : kStagesFit;
  static constexpr bool kQSmem = kO > 32;             // Q fragments re-read from shared memory
  static constexpr int kRing = kWarps * kStages * kTile;
  static constexpr int kQBytes = kQSmem ? 8 * NT * D * 2 : 0;
  static constexpr int kRl = kWarps * 8 * NT * 16;    // the warps' references and sums
  static constexpr int kSc = kWarps * kStages * 8;    // a staged tile's scales
  static constexpr int kBytes = kRing + kQBytes + kRl + kSc + (kWarps + 2) * 8;
  static_assert(kWarps / 2 * 8 * NT * D * 4 <= kRing, "the merge reuses the ring");
};

// What turns sum_i w_i V_i into the output: 2^(r - 7 - c) over the sum (0 where nothing was seen), as two
// factors, since the power alone may leave fp32's range (values' scales near either end of E8M0's) where
// the output does not.
__device__ __forceinline__ float2 pa_factor(float ref, float top, float sum) {
  const float e = ref - top - 7.f, half = 0.5f * e;
  return sum == 0.f ? make_float2(0.f, 0.f) : make_float2(ex2_approx(half) / sum, ex2_approx(e - half));
}

// out[8 dims] of one column from 8 consecutive values.
template <bool F16>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(Act<F16>::pack(v[0], v[1]), Act<F16>::pack(v[2], v[3]), Act<F16>::pack(v[4], v[5]),
                    Act<F16>::pack(v[6], v[7]));
}

template <bool F16, int D, int NT>
__global__ void __launch_bounds__(32 * PaShape<D, NT>::kWarps, PaShape<D, NT>::kCtas) paged_attn_kernel(const PagedAttnArgs a) {
  using P = PaShape<D, NT>;
  using T = typename Act<F16>::T;
  constexpr int W = P::kWarps, S = P::kStages, KS = D / 16;
  extern __shared__ __align__(128) uint8_t pa_smem[];
  uint2* q_sm = reinterpret_cast<uint2*>(pa_smem + P::kRing);
  float4* rl_sm = reinterpret_cast<float4*>(pa_smem + P::kRing + P::kQBytes);
  float2* sc_sm = reinterpret_cast<float2*>(pa_smem + P::kRing + P::kQBytes + P::kRl) + (threadIdx.x >> 5) * S;
  long long* plan_sm = reinterpret_cast<long long*>(pa_smem + P::kRing + P::kQBytes + P::kRl + P::kSc);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  uint8_t* ring_p = pa_smem + warp * S * P::kTile;
  const uint32_t ring = smem_u32(ring_p);
  const int kvh = a.cache.kv_heads, group = a.heads / kvh, page = a.cache.page, block = a.cache.block;
  const int kap = pa_kappa(g);

  pdl_wait();
  pdl_launch();
  if (tid == 0 && !a.whole) a.split[blockIdx.x].pieces = 0;
  const Share sh = find_share<NT, W>(a, blockIdx.x, gridDim.x, plan_sm);
  if (sh.seq < 0) return;
  // Where the share stands lies in shared memory between pieces, not in registers: the sequence, the
  // unit in it, the units left.
  if (tid == 0) plan_sm[0] = sh.seq, plan_sm[1] = sh.first - sh.seq0, plan_sm[2] = sh.last - sh.first, plan_sm[3] = sh.per;
  for (bool first_piece = true;; first_piece = false) {
    __syncthreads();
    int seq = (int)plan_sm[0];
    long long at = plan_sm[1];
    const long long left = plan_sm[2];
    if (left <= 0) break;
    SeqWork w = seq_work<NT, W>(a, seq);
    while (at >= w.units) {
      at -= w.units;
      w = seq_work<NT, W>(a, ++seq);
    }
    // this piece: kv head hk, column tile ct, steps [step0, step1)
    const int item = (int)(a.whole ? at : at / w.steps), step0 = a.whole ? 0 : (int)(at % w.steps);
    const int step1 = a.whole ? w.steps : (int)min((long long)w.steps, step0 + left);
    const int ct = item % w.cts, hk = item / w.cts;
    const int col0 = ct * 8 * NT;
    // what its first and last row see
    const int j0 = col0 / group, j1 = (min(col0 + 8 * NT, w.cols) - 1) / group;
    const int cap = a.rows.width * page;
    const int vis0 = w.end - w.n + 1;
    auto vis = [&](int j) { return vis0 + j; };
    auto low = [&](int j) { return window_low(vis(j), a.window); };
    const int any_lo = low(j0), any_hi = min(vis(j1), cap), all_lo = low(j1), all_hi = min(vis(j0), cap);

    // Q: column n's dims 64 c + 16 t + 4 q + {0 .. 3} are step 4 c + q's fragment of lane (n, t)
    uint32_t qf[P::kQSmem ? 1 : NT][P::kQSmem ? 1 : KS][2];
    float qmul[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int col = col0 + 8 * n + g;
      uint32_t raw[KS][2];
      float amax = 0.f;
      const T* qp = reinterpret_cast<const T*>(a.q) + (w.row0 + col / group) * a.q_ld + (hk * group + col % group) * D;
      if (!P::kQSmem || warp == n % W) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          uint4 x[2] = {};
          if (col < w.cols) {
            x[0] = ldg16(qp + 64 * c + 16 * t);
            x[1] = ldg16(qp + 64 * c + 16 * t + 8);
          }
          const uint32_t v[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            raw[4 * c + i / 2][i & 1] = v[i];
            if (!F16) {
              const float2 f = Act<F16>::unpack(v[i]);
              amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
          }
        }
      }
      float inv = 1.f;
      if (!F16) {
        // scale the column so that its largest value is below 2^14
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        int e = (int)((__float_as_uint(amax) >> 23) & 255);
        e = e == 255 ? 127 + 13 : max(e, 40);
        const float mul = __uint_as_float((uint32_t)(254 + 13 - e) << 23);
        inv = __uint_as_float((uint32_t)(e - 13) << 23);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 f = Act<F16>::unpack(raw[k][i]);
            raw[k][i] = pack_f16x2(f.x * mul, f.y * mul);
          }
      }
      if (P::kQSmem) {
        if (warp == n % W) {
#pragma unroll
          for (int k = 0; k < KS; ++k) q_sm[(n * KS + k) * 32 + lane] = make_uint2(raw[k][0], raw[k][1]);
          if (t == 0) rl_sm[8 * n + g].x = inv;
        }
      } else {
#pragma unroll
        for (int k = 0; k < KS; ++k) qf[n][k][0] = raw[k][0], qf[n][k][1] = raw[k][1];
        qmul[n][0] = __shfl_sync(0xffffffffu, inv, 8 * t) * a.scale;
        qmul[n][1] = __shfl_sync(0xffffffffu, inv, 8 * t + 4) * a.scale;
      }
    }
    if (P::kQSmem) {
      __syncthreads();
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) qmul[n][e] = rl_sm[8 * n + 2 * t + e].x * a.scale;
    }

    float o[NT][KS][4], ref[NT][2], top[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
      ref[n][0] = ref[n][1] = top[n][0] = top[n][1] = -FLT_MAX;
      l[n][0] = l[n][1] = 0.f;
    }

    // the warp's tiles: w.tile0 + first + W j, j < count
    const int first = step0 * W + warp;
    const int count = max(0, (min(step1 * W, w.tiles) - first + W - 1) / W);
    // lane i holds of tile 32 b + i of the batch b being issued where its keys begin in the cache, or -1 where
    // the piece sees none of its tokens, and its scales (the keys' power of two, the values' exponent), which
    // it leaves beside the staged tile. The divisions by the page and the block are made here, once a tile by
    // one lane.
    int64_t bat_at = -1;
    float2 bat_sc = make_float2(0.f, 0.f);
    const int tile_first = w.tile0 + first;
    auto load_batch = [&](int b) {
      const int j = 32 * b + lane, p0 = (tile_first + W * j) * 16;
      bat_at = -1;
      bat_sc.x = 0.f;  // no tile
      if (j < count && p0 < any_hi && p0 + 16 > any_lo) {
        const int pg = token_page(a.rows, a.cache, seq, p0);
        if (pg >= 0) {
          const int off = p0 % page;
          const int64_t head = (int64_t)pg * kvh + hk, ci = head * (page / block) + off / block;
          bat_at = (head * page + off) * D;
          bat_sc = make_float2(pow2c(a.cache.k_codes[ci]), (float)((int)a.cache.v_codes[ci] - 127));
        }
      }
    };
    const uint32_t lane_dst = ring + pa_chunk<D>(lane / (D / 16), lane % (D / 16));
    int is_st = 0;  // the stage to issue into
    auto issue = [&](int j) {
      if (j < count) {
        if (j % 32 == 0) load_batch(j / 32);
        const int64_t at = __shfl_sync(0xffffffffu, bat_at, j & 31);
        if (lane == (j & 31)) sc_sm[is_st] = bat_sc;
        if (at >= 0) {
          const uint8_t *ks = a.cache.k + at + lane * 16, *vs = a.cache.v + at + lane * 16;
          const uint32_t dst = is_st * P::kTile;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            // 32 pieces on are 512 / D rows on: so many units further round the swizzle
            const uint32_t d = (lane_dst ^ (D == 64 ? 0 : (512 / D * i & 7) << 4)) + dst + i * 512;
            cp_async16_stream(d, ks + i * 512);
            cp_async16_stream(d + 16 * D, vs + i * 512);
          }
        }
        is_st = is_st == S - 1 ? 0 : is_st + 1;
      }
      cp_async_commit();
    };
#pragma unroll 1
    for (int j = 0; j < S - 1; ++j) issue(j);
    int rd_st = 0;  // the stage to read
#pragma unroll 1
    for (int j = 0; j < count; ++j) {
      issue(j + S - 1);
      cp_async_wait<S - 1>();
      __syncwarp();
      const uint8_t *kt = ring_p + rd_st * P::kTile, *vt = kt + 16 * D;
      const float2 sc = sc_sm[rd_st];
      rd_st = rd_st == S - 1 ? 0 : rd_st + 1;
      if (sc.x == 0.f) continue;
      const float ks = sc.x, ev = sc.y;
      const int p0 = (tile_first + W * j) * 16;
      const bool edge = p0 < all_lo || p0 + 16 > all_hi;

      // S^T = K Q^T
      // (QC chains a column tile: one tensor-core instruction waits for the one before it in its chain)
      constexpr int QC = NT <= 2 ? 2 : 1;
      float sq[QC][NT][4];
#pragma unroll
      for (int x = 0; x < QC; ++x)
#pragma unroll
        for (int n = 0; n < NT; ++n) sq[x][n][0] = sq[x][n][1] = sq[x][n][2] = sq[x][n][3] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const uint4 x = pa_lds<uint4>(kt + pa_chunk<D>(kap, 4 * c + t));
        const uint4 y = pa_lds<uint4>(kt + pa_chunk<D>(kap + 8, 4 * c + t));
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t a0, a1, a2, a3;
          e4m3x4_f16(xs[i], a0, a2);
          e4m3x4_f16(ys[i], a1, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint2 b;
            if (P::kQSmem) b = q_sm[(n * KS + 4 * c + i) * 32 + lane];
            else b = make_uint2(qf[P::kQSmem ? 0 : n][P::kQSmem ? 0 : 4 * c + i][0],
                                qf[P::kQSmem ? 0 : n][P::kQSmem ? 0 : 4 * c + i][1]);
            pa_mma(sq[i % QC][n], a0, a1, a2, a3, b.x, b.y);
          }
        }
      }

      float(&s)[NT][4] = sq[0];
#pragma unroll
      for (int x = 1; x < QC; ++x)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] += sq[x][n][e];

      // s: scores, base 2; elements (token kappa, column 2t), (kappa, 2t + 1), (kappa + 8, ..)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] *= qmul[n][e & 1] * ks;
      if (edge) {
        int c0 = col0 + 2 * t;
        asm volatile("" : "+r"(c0));  // nothing of this branch is to be kept in registers from tile to tile
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int j = (c0 + 8 * n + e) / group, hi = min(vis(j), cap), lo = low(j), p = p0 + kap;
            if (p >= hi || p < lo) s[n][e] = -INFINITY;
            if (p + 8 >= hi || p + 8 < lo) s[n][e + 2] = -INFINITY;
          }
      }
      // how far the scores lie above where the references stand (at most 2^8 and 2^60 are let pass)
      float far = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          far = fmaxf(far, fmaxf(s[n][e], s[n][e + 2]) - fminf(ref[n][e] + (8.f - ev), top[n][e] + 60.f));
      if (__any_sync(0xffffffffu, far > 0.f)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float m = fmaxf(s[n][e], s[n][e + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            const float r = fmaxf(m + ev, ref[n][e]), f = ex2_approx(ref[n][e] - r);
            m = fmaxf(m, top[n][e]);
            l[n][e] *= ex2_approx(top[n][e] - m);
            ref[n][e] = r;
            top[n][e] = m;
#pragma unroll
            for (int i = 0; i < KS; ++i) o[n][i][e] *= f, o[n][i][e + 2] *= f;
          }
      }
      uint32_t ph[NT][2], pl[NT][2];  // the weights' f16 heads, and what those leave
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) l[n][e] += ex2_approx(s[n][e] - top[n][e]) + ex2_approx(s[n][e + 2] - top[n][e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = ex2_approx(s[n][e] + (ev + 7.f - ref[n][e & 1]));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = s[n][2 * e], y = s[n][2 * e + 1];
          const uint32_t head = cvt_f16x2(x, y);
          const float2 h = Act<true>::unpack(head);
          ph[n][e] = movmatrix(head);
          pl[n][e] = movmatrix(cvt_f16x2(x - h.x, y - h.y));
        }
      }

      // O^T += V^T P^T: lane (g, t) reads tokens t, 7 - t, t + 8, 15 - t (kappa of the mma's k = 2t,
      // 2t + 1, 2t + 8, 2t + 9) of its D / 8 dims; dims 2 i and 2 i + 1 are M tile i's rows g, g + 8
      uint32_t v[4][D / 32];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = ((r & 1) ? 7 - t : t) + (r >> 1) * 8;
        if (D == 64) {
          const uint2 x = pa_lds<uint2>(vt + pa_chunk<D>(row, g >> 1) + (g & 1) * 8);
          v[r][0] = x.x, v[r][1] = x.y;
        } else {
#pragma unroll
          for (int c = 0; c < D / 128; ++c) {
            const uint4 x = pa_lds<uint4>(vt + pa_chunk<D>(row, 8 * c + ((g >> 1) | (g & 1) << 2)));
            v[r][4 * c] = x.x, v[r][4 * c + 1] = x.y, v[r][4 * c + 2] = x.z, v[r][4 * c + 3] = x.w;
          }
        }
      }
      bool nan = false;
      if (edge) {
        // tokens that no row of the piece sees hold anything; NaN in one that only some rows see must not
        // reach the others as 0 NaN, so NaN bytes go in as zeros here and come back below
        int p1 = p0;
        asm volatile("" : "+r"(p1));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int p = p1 + ((r & 1) ? 7 - t : t) + (r >> 1) * 8;
          const bool seen = p >= any_lo && p < any_hi;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            const uint32_t m = nan_bytes(v[r][i]);
            nan |= seen && m;
            v[r][i] = seen ? v[r][i] & ~m : 0u;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t a0, a1, a2, a3;
          const uint32_t sel = h ? 0x7362 : 0x5140;  // (x_2h, y_2h, x_2h+1, y_2h+1)
          e4m3x4_f16(__byte_perm(v[0][i], v[1][i], sel), a0, a1);
          e4m3x4_f16(__byte_perm(v[2][i], v[3][i], sel), a2, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) pa_mma(o[n][2 * i + h], a0, a1, a2, a3, ph[n][0], ph[n][1]);
#pragma unroll
          for (int n = 0; n < NT; ++n) pa_mma(o[n][2 * i + h], a0, a1, a2, a3, pl[n][0], pl[n][1]);
        }
      if (edge && __any_sync(0xffffffffu, nan)) {
        // this lane's dims of each token again: what holds NaN makes NaN of the columns that see it
#pragma unroll 1
        for (int r = 0; r < 16; ++r) {
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            const uint8_t* x = D == 64 ? vt + pa_chunk<D>(r, g >> 1) + (g & 1) * 8 + 4 * i
                                       : vt + pa_chunk<D>(r, 8 * (i / 4) + ((g >> 1) | (g & 1) << 2)) + 4 * (i & 3);
            const uint32_t m = nan_bytes(pa_lds<uint32_t>(x));
            if (!m) continue;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int j = (col0 + 8 * n + 2 * t + e) / group;
                if (p0 + r >= min(vis(j), cap) || p0 + r < low(j)) continue;
                const float bad = __uint_as_float(0x7fffffffu);
                if (m & 0xffu) o[n][2 * i][e] = bad;
                if (m & 0xff00u) o[n][2 * i][e + 2] = bad;
                if (m & 0xff0000u) o[n][2 * i + 1][e] = bad;
                if (m & 0xff000000u) o[n][2 * i + 1][e + 2] = bad;
              }
          }
        }
      }
      __syncwarp();
    }

    // join the warps: the largest reference of each column, then O and l by a tree
    cp_async_wait<0>();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
    __syncthreads();
    if (g == 0)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) rl_sm[warp * 8 * NT + 8 * n + 2 * t + e] = make_float4(ref[n][e], top[n][e], l[n][e], 0.f);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float m = -FLT_MAX, c = -FLT_MAX, sum = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float4 x = rl_sm[i * 8 * NT + 8 * n + 2 * t + e];
          m = fmaxf(m, x.x);
          c = fmaxf(c, x.y);
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float4 x = rl_sm[i * 8 * NT + 8 * n + 2 * t + e];
          sum = fmaf(x.z, ex2_approx(x.y - c), sum);
        }
        const float f = ex2_approx(ref[n][e] - m);
#pragma unroll
        for (int i = 0; i < KS; ++i) o[n][i][e] *= f, o[n][i][e + 2] *= f;
        ref[n][e] = m;
        top[n][e] = c;
        l[n][e] = sum;
      }
    float4* mb = reinterpret_cast<float4*>(pa_smem);
#pragma unroll
    for (int n_w = W; n_w > 1; n_w = (n_w + 1) / 2) {
      const int half = (n_w + 1) / 2;
      if (warp >= half && warp < n_w)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < KS; ++i)
            mb[(((warp - half) * NT + n) * KS + i) * 32 + lane] =
                make_float4(o[n][i][0], o[n][i][1], o[n][i][2], o[n][i][3]);
      __syncthreads();
      if (warp < n_w - half)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            const float4 x = mb[((warp * NT + n) * KS + i) * 32 + lane];
            o[n][i][0] += x.x, o[n][i][1] += x.y, o[n][i][2] += x.z, o[n][i][3] += x.w;
          }
      __syncthreads();
    }
    const bool whole = step0 == 0 && step1 == w.steps;
    const int slot = 2 * blockIdx.x + (first_piece ? 0 : 1);
    if (tid == 0 && step0 == 0 && !whole) {
      const long long per = plan_sm[3];
      a.split[blockIdx.x] = {1 + (int)((w.steps - step1 + per - 1) / per), slot, w.row0, hk * group, col0, w.cols};
    }
    if (warp == 0)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = 8 * n + 2 * t + e, col = col0 + c;
          if (col >= w.cols) continue;
          const int j = col / group, h = hk * group + col % group;
          // this lane's dims: D / 8 from d0 on (D = 256: two runs of 16, 128 apart)
          const int d0 = D == 64 ? 8 * g : 16 * ((g >> 1) | (g & 1) << 2);
          if (whole) {
            float sum = l[n][e];
            if (a.sink) sum += ex2_approx(a.sink[h] * 1.44269504f - top[n][e]);
            const float2 f = pa_factor(ref[n][e], top[n][e], sum);
            T* y = reinterpret_cast<T*>(a.out) + (w.row0 + j) * a.out_ld + h * D;
#pragma unroll
            for (int i = 0; i < KS / 4; ++i) {
              float x[8];
#pragma unroll
              for (int b = 0; b < 8; ++b) x[b] = o[n][4 * i + b / 2][e + 2 * (b & 1)] * f.x * f.y;
              *reinterpret_cast<uint4*>(y + (i / 2) * 128 + d0 + (i & 1) * 8) = pack8<F16>(x);
            }
          } else {
            if (g == 0) a.part_rl[(int64_t)slot * 8 * NT + c] = make_float4(ref[n][e], top[n][e], l[n][e], 0.f);
            float* y = a.part + ((int64_t)slot * 8 * NT + c) * D;
#pragma unroll
            for (int i = 0; i < KS / 2; ++i) {
              const float4 x = make_float4(o[n][2 * i][e], o[n][2 * i][e + 2], o[n][2 * i + 1][e], o[n][2 * i + 1][e + 2]);
              *reinterpret_cast<float4*>(y + (i / 4) * 128 + d0 + (i & 3) * 4) = x;
            }
          }
        }
    const int used = a.whole ? 1 : step1 - step0;
    if (tid == 0) plan_sm[0] = seq, plan_sm[1] = at + used, plan_sm[2] = left - used;
  }
}

constexpr int kPaJoinThreads = 128;

// Join the pieces of the item that begins in share blockIdx.x and goes on past its end (at most one): one
// CTA a column. The pieces are summed D / 4 threads a piece, several at a time, and those sums in order.
template <bool F16, int D, int NT>
__global__ void __launch_bounds__(kPaJoinThreads) paged_join_kernel(const PagedAttnArgs a) {
  using T = typename Act<F16>::T;
  constexpr int LG = D / 4, PG = kPaJoinThreads / LG;  // threads a piece, pieces at a time
  __shared__ float red[3][kPaJoinThreads / 32];
  __shared__ float4 sums[PG][LG];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = blockIdx.y;
  pdl_wait();
  const PaSplit sp = a.split[blockIdx.x];
  if (!sp.pieces || sp.col0 + c >= sp.cols) return;
  auto at = [&](int i) { return (int64_t)(i ? 2 * ((int)blockIdx.x + i) : sp.slot) * 8 * NT + c; };
  float m = -FLT_MAX, top = -FLT_MAX, sum = 0.f;
  for (int i = tid; i < sp.pieces; i += kPaJoinThreads) {
    const float4 rl = a.part_rl[at(i)];
    m = fmaxf(m, rl.x);
    top = fmaxf(top, rl.y);
  }
  m = warp_max(m), top = warp_max(top);
  if (lane == 0) red[0][warp] = m, red[1][warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPaJoinThreads / 32; ++w) m = fmaxf(m, red[0][w]), top = fmaxf(top, red[1][w]);
  for (int i = tid; i < sp.pieces; i += kPaJoinThreads) {
    const float4 rl = a.part_rl[at(i)];
    sum = fmaf(rl.z, ex2_approx(rl.y - top), sum);
  }
  sum = warp_sum(sum);
  if (lane == 0) red[2][warp] = sum;
  const int d = tid % LG, pg = tid / LG;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = pg; i < sp.pieces; i += PG) {
    const float f = ex2_approx(a.part_rl[at(i)].x - m);
    const float4 y = *reinterpret_cast<const float4*>(a.part + at(i) * D + 4 * d);
    o.x = fmaf(y.x, f, o.x), o.y = fmaf(y.y, f, o.y), o.z = fmaf(y.z, f, o.z), o.w = fmaf(y.w, f, o.w);
  }
  sums[pg][d] = o;
  __syncthreads();
  if (pg) return;
#pragma unroll
  for (int i = 1; i < PG; ++i) {
    const float4 y = sums[i][d];
    o.x += y.x, o.y += y.y, o.z += y.z, o.w += y.w;
  }
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kPaJoinThreads / 32; ++w) sum += red[2][w];
  const int col = sp.col0 + c, group = a.heads / a.cache.kv_heads, h = sp.h0 + col % group;
  if (a.sink) sum += ex2_approx(a.sink[h] * 1.44269504f - top);
  const float2 f = pa_factor(m, top, sum);
  T* y = reinterpret_cast<T*>(a.out) + (int64_t)(sp.row0 + col / group) * a.out_ld + h * D + 4 * d;
  *reinterpret_cast<uint2*>(y) = make_uint2(Act<F16>::pack(o.x * f.x * f.y, o.y * f.x * f.y),
                                            Act<F16>::pack(o.z * f.x * f.y, o.w * f.x * f.y));
}

}  // namespace dsv41
