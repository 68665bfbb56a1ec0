// Products of a few rows with 4-bit weights and group scales:
//
//   y[m, n] = sum_k x[m, k] (q[n, k] - z[n, k / G]) s[n, k / G]
//           = sum_g s[n, g] ( sum_{k in g} x[m, k] q[n, k]  -  z[n, g] sum_{k in g} x[m, k] )
//
// q packed two to a byte, the even k in the low nibble; z = 8 where not given.
//
// Bound by HBM: each weight is read once for all rows of x.  At HBM rate an SM
// has to take in some 46 weights a cycle and can issue 128 lanes of
// instructions, so the unpacking decides.  The products run on mma.sync
// m16n8k16 with 16 rows of q as the A operand and the rows of x as its 8
// columns.  (tcgen05 takes its operands from shared memory or TMEM: the
// unpacked weights, four times the bytes, would have to be written there
// first.)  The A operand is made with 5 instructions per 8 weights:
// as fp16 bits, word & 0x000F000F is the pair (q0, q4) times 2^-24 and
// word & 0x00F000F0 the pair (q1, q5) times 2^-20 -- subnormal numbers, which
// the tensor core multiplies exactly -- and the same masks on word >> 8 give
// (q2, q6) and (q3, q7).  One MMA takes the 2^-24 pairs, one the 2^-20 pairs,
// into accumulators of their own; the powers of two leave with the group's
// scale.  k may be summed in any order, so nothing is shuffled: the pairs of
// x are permuted to match once, as x is staged in shared memory.
// (As 128 + q in bf16, minus 136, with x permuted on every use and every loop
// unrolled, 3 x 100003 x 5120 took 92 us; it takes 62.6, 4.2 TB/s.  1 x 4096 x
// 4096 takes 5.8 us, of it some 3 the latency of a launch, staging x and one
// chain of groups; 8 x 14336 x 4096 with zero points and groups of 64 22.8: x is
// staged once by each CTA, and the two sums of a group cost as much as its MMAs.)
//
// x is staged as fp16 whatever its type: each group of a row is scaled by a
// power of two that brings its largest value to [2^14, 2^15), so 16-bit
// inputs keep every bit down to 2^-29 of that value and lose at most 2^-40 of
// it below; fp32 is split into three such planes (2^-33 of the largest value
// is left out) and meets q - 8 as normal numbers (q4_pair).  The scale and
// sum_{k in g} x, in fp32, stand beside it.  Infinities and NaN would meet their
// own sum (inf - z inf) and numbers past 2^120 overflow it: a CTA that staged such
// a number does the outputs of that row again at the end, from the definition.
//
// The warps of a CTA split k; their partial sums meet in shared memory in
// warp order.  A CTA walks over row tiles with the next weights always in
// flight, and where x does not fit, over chunks of k outside that, with the
// tiles' sums kept in shared memory.  With few row tiles the CTAs of a
// cluster split k again and add up in rank order.
#pragma once

#include "molten/common.cuh"

namespace molten {

struct Q4Args {
  const void* x;                   // [m, k], rows x_stride elements apart
  const uint8_t* q;                // [n, k/2]
  const void* scales;              // [n, k/G]
  const void* zeros;               // [n, k/G] or null
  void* out;                       // [m, n]
  long long x_stride, n;
  int m, k;
  int warps_n_log;                 // log2 of the warps along the rows of q (of the CTA's)
  int ksplit_log;                  // log2 of the CTAs of the cluster, along k
  int chunk;                       // groups of k staged at once
  int tiles;                       // row tiles of 16 * warps_n
  int teams;                       // CTAs (clusters) that share the tiles
  int reserved;
};

__device__ __forceinline__ void q4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                       uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
               "{%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The nibbles at bits AT and AT + 16 of a word as a pair of halves: q 2^-24
// (AT = 0) or q 2^-20 (AT = 4), subnormal, by one mask.  EXACT: q - 8 or
// 16 (q - 8) as normal numbers, by an or and a packed subtraction more: the
// tensor core lines products up by the operands' exponent fields, so a
// subnormal operand's sums keep some 19 bits (measured: 1.4e-6 of the result,
// far below a 16-bit output's rounding, but not below an fp32 one's).
template <int AT, bool EXACT>
__device__ __forceinline__ uint32_t q4_pair(uint32_t word) {
  const uint32_t v = word & (0x000F000Fu << AT);
  if constexpr (!EXACT) return v;
  const uint32_t u = v | 0x64006400u;                // 1024 + q, 1024 + 16 q
  const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&u),
                            __float2half2_rn(AT ? 1152.0f : 1032.0f));
  return *reinterpret_cast<const uint32_t*>(&d);
}

// W consecutive 32-bit words (W = 4, 2, 1: 16, 8, 4 bytes).  A lane's 4-byte
// loads leave half of each sector for the next group's, so those go through
// L1; wider ones are read once.
template <int W>
__device__ __forceinline__ void q4_load(const uint8_t* p, uint32_t (&w)[W]) {
  if constexpr (W == 4) {
    const uint4 v = ld16<kLoadStream>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (W == 2) {
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v2.u32 {%0,%1}, [%2];"
                 : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  } else {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
}

// d = a b, the accumulators starting at zero
__device__ __forceinline__ void q4_mma0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
               "{%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint4 q4_lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float2 q4_lds8(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}

// Shared memory: x as [word of the lane][group][row][lane of the quad] slots
// of 8 halves (pairs (0,4) (2,6) (1,5) (3,7)) per plane, one zero slot, then
// (sum of x, scale) per [group][row], the warps' partial sums (two buffers)
// and the sums of the CTA's tiles.
template <int G, int NT, int PLANES, int WARPS>
struct Q4Smem {
  static constexpr int W = G / 32, RED = NT * 128;   // partial sums of one warp
  uint4* xs;
  float2* gs;
  float* red;
  float* sums;
  int word, plane;                                   // (group, row)s; slots of a plane
  __device__ __forceinline__ Q4Smem(uint8_t* raw, const Q4Args& a) {
    word = a.chunk * a.m;
    plane = word * 4 * W;
    xs = reinterpret_cast<uint4*>(raw);
    gs = reinterpret_cast<float2*>(xs + PLANES * plane + 1);
    red = reinterpret_cast<float*>(gs + a.chunk * a.m);
    sums = red + 2 * WARPS * RED;
  }
};

// An infinity, a NaN, or so large that the sum of a group could pass the range.
__device__ __forceinline__ bool q4_wild(float x) { return !(fabsf(x) < 1.329227995784916e36f); }   // 2^120

// Stage groups [g0, g0 + count) of every row of x: a group of a row to G/8
// lanes, STEP groups' loads in flight at once.  True: a group holds what q4_wild
// says.
template <typename XT, int G, int NT, int PLANES, int WARPS>
__device__ __forceinline__ bool q4_stage(const Q4Args& a, const Q4Smem<G, NT, PLANES, WARPS>& s,
                                         int g0, int count) {
  constexpr int W = G / 32, LANES = G / 8;
  constexpr int STEP = NT == 1 ? 2 : 4, UNITS = WARPS * 32 / LANES;
  const int unit = threadIdx.x / LANES, l = threadIdx.x % LANES;
  const int t = l / W, w = l % W;
  const int total = count * a.m;
  const XT* x = static_cast<const XT*>(a.x) + (long long)g0 * G + 8 * l;
  int row = unit / count, grp = unit - row * count;  // of the next load
  bool wild = false;
#pragma unroll 1
  for (int base = 0; base < total; base += UNITS * STEP) {   // (whole warps shuffle)
    Slot<XT, 8> v[STEP];
    int at[STEP];                                    // group * m + row, or -1
#pragma unroll
    for (int j = 0; j < STEP; ++j) {
      at[j] = row < a.m ? grp * a.m + row : -1;
      v[j] = load_slot<kLoadDefault, XT, 8>(x + min(row, a.m - 1) * a.x_stride + (long long)grp * G);
      grp += UNITS;
      while (grp >= count) { grp -= count; ++row; }
    }
#pragma unroll
    for (int j = 0; j < STEP; ++j) {
      float f[8], top = 0.0f, sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = to_f32(v[j].v[e]);
        top = fmaxf(top, fabsf(f[e]));
        sum += f[e];
      }
#pragma unroll
      for (int d = LANES / 2; d >= 1; d /= 2) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        sum += __shfl_xor_sync(0xffffffffu, sum, d);
      }
      wild |= q4_wild(top) || sum != sum;            // (the maximum with NaN is the other)
      // up = 2^(14 - exponent of top), its bits made directly; e is kept where
      // up and its reciprocal are normal numbers
      int e = (int)(__float_as_uint(top) >> 23);
      e = e < 40 ? 40 : (e > 254 ? 254 : e);
      const float up = __uint_as_float((uint32_t)(268 - e) << 23);
      if (at[j] < 0) continue;
      if (l == 0) {
        // the products come as x up q 2^-24 (EXACT: x up (q - 8)); the group's
        // scale takes the 2^24, so the sum of x goes without it
        s.gs[at[j]] = make_float2(sum * (PLANES == 3 ? 1.0f : 5.9604645e-8f),
                                  __uint_as_float((uint32_t)(e - 14) << 23));
      }
      uint4* dst = s.xs + (w * s.word + at[j]) * 4 + t;
#pragma unroll
      for (int q = 0; q < 8; ++q) f[q] *= up;
#pragma unroll
      for (int pl = 0; pl < PLANES; ++pl) {
        const __half2 h0 = __floats2half2_rn(f[0], f[4]), h1 = __floats2half2_rn(f[2], f[6]);
        const __half2 h2 = __floats2half2_rn(f[1], f[5]), h3 = __floats2half2_rn(f[3], f[7]);
        dst[pl * s.plane] = make_uint4(*reinterpret_cast<const uint32_t*>(&h0),
                                       *reinterpret_cast<const uint32_t*>(&h1),
                                       *reinterpret_cast<const uint32_t*>(&h2),
                                       *reinterpret_cast<const uint32_t*>(&h3));
        if (pl + 1 < PLANES) {                       // what the plane leaves, exactly
          f[0] -= __low2float(h0); f[4] -= __high2float(h0);
          f[2] -= __low2float(h1); f[6] -= __high2float(h1);
          f[1] -= __low2float(h2); f[5] -= __high2float(h2);
          f[3] -= __low2float(h3); f[7] -= __high2float(h3);
        }
      }
    }
  }
  return wild;
}

// The rows of x that hold a wild number, with the rows of q of this team's
// tiles, over all of k in 64 bits: a warp to an output.
template <typename XT, typename ST, typename OT, int G, bool ZEROS, int WARPS>
__device__ __noinline__ void q4_wild_rows(const Q4Args& a, int team) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long groups = a.k / G;
#pragma unroll 1
  for (int row = 0; row < a.m; ++row) {
    const XT* x = static_cast<const XT*>(a.x) + row * a.x_stride;
    bool wild = false;
#pragma unroll 1
    for (int k = lane; k < a.k; k += 32) wild |= q4_wild(to_f32(x[k]));
    if (!__any_sync(0xffffffffu, wild)) continue;
#pragma unroll 1
    for (int tile = team; tile < a.tiles; tile += a.teams) {
#pragma unroll 1
      for (int i = warp; i < 16 << a.warps_n_log; i += WARPS) {
        const long long n = ((long long)tile << a.warps_n_log) * 16 + i;
        if (n >= a.n) break;
        double y = 0.0;
#pragma unroll 1
        for (int b = lane; b < a.k / 2; b += 32) {   // a byte of q: two k of one group
          const int two = a.q[n * (a.k / 2) + b];
          const long long g = n * groups + 2 * b / G;
          double z = 8.0;
          if constexpr (ZEROS) z = (double)to_f32(static_cast<const ST*>(a.zeros)[g]);
          const double s = (double)to_f32(static_cast<const ST*>(a.scales)[g]);
          y += (double)to_f32(x[2 * b]) * ((double)(two & 15) - z) * s;
          y += (double)to_f32(x[2 * b + 1]) * ((double)(two >> 4) - z) * s;
        }
#pragma unroll
        for (int d = 16; d >= 1; d /= 2) y += __shfl_xor_sync(0xffffffffu, y, d);
        if (lane == 0) static_cast<OT*>(a.out)[row * a.n + n] = from_f32<OT>((float)y);
      }
    }
  }
}

__device__ __forceinline__ void q4_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\t"
               "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// NT: blocks of 8 rows of x.  G: group size.  DEPTH: groups in flight a warp.
template <typename XT, typename ST, typename OT, int G, int NT, bool ZEROS, int DEPTH, int WARPS>
__device__ __forceinline__ void q4_matvec(const Q4Args& a, uint8_t* raw) {
  constexpr int PLANES = std::is_same<XT, float>::value ? 3 : 1;
  constexpr bool EXACT = PLANES == 3;                // zero points count from 8
  constexpr int W = G / 32;                          // words per lane, row and group
  typedef Q4Smem<G, NT, PLANES, WARPS> Smem;
  const Smem sm(raw, a);
  constexpr int RED = Smem::RED;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane / 4, t = lane % 4;
  const int warps_n = 1 << a.warps_n_log, wn = warp & (warps_n - 1), wk = warp >> a.warps_n_log;
  const int warps_k = WARPS >> a.warps_n_log, ksplit = 1 << a.ksplit_log;
  const int team = blockIdx.x >> a.ksplit_log, rank = blockIdx.x & (ksplit - 1);
  const uint32_t groups = (uint32_t)a.k / G;         // (below 2^26)
  // groups of this CTA, walked in chunks
  const int cta0 = (int)(groups * rank >> a.ksplit_log);
  const int cta1 = (int)(groups * (rank + 1) >> a.ksplit_log);
  const int per = warps_n * 16 * a.m;                // sums of one tile
  if (threadIdx.x == 0) sm.xs[PLANES * sm.plane] = make_uint4(0u, 0u, 0u, 0u);

  // this lane's slots of x (rows past m: the zero slot, without a stride) and
  // (sum, scale) pairs of its two columns
  const uint32_t xs0 = static_cast<uint32_t>(__cvta_generic_to_shared(sm.xs));
  const uint32_t gs0 = static_cast<uint32_t>(__cvta_generic_to_shared(sm.gs));
  uint32_t xa[NT], ga[NT][2];
  const uint32_t x_word = (uint32_t)sm.word * 64u;   // bytes from one word to the next
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int row = i * 8 + g;
    xa[i] = row < a.m ? xs0 + (uint32_t)(row * 4 + t) * 16u : 0u;
#pragma unroll
    for (int e = 0; e < 2; ++e) ga[i][e] = gs0 + 8u * (uint32_t)min(i * 8 + 2 * t + e, a.m - 1);
  }
  const uint32_t zero_slot = xs0 + (uint32_t)(PLANES * sm.plane) * 16u;
  // the sum that this thread adds up at the end of a tile
  const int my_on = threadIdx.x / (16 * a.m), my_rest = threadIdx.x - my_on * (16 * a.m);

  int wild = 0;                                      // (the same in every thread)
  for (int c0 = cta0; c0 < cta1; c0 += a.chunk) {
    const int count = min(a.chunk, cta1 - c0);
    // this warp's groups of the chunk, the same of every tile
    const int l0 = (int)((uint32_t)count * wk * warps_n / WARPS);
    const int gk = (int)((uint32_t)count * (wk + 1) * warps_n / WARPS) - l0;

    uint32_t w0[DEPTH][W], w1[DEPTH][W];
    ST sc[DEPTH][2], zr[DEPTH][2];
    int f_tile = team, f_left = 0;                   // next tile to fetch, groups left of it
    const uint8_t *q0 = nullptr, *q1 = nullptr;
    const ST *s0 = nullptr, *s1 = nullptr, *z0 = nullptr, *z1 = nullptr;
    const uint8_t* q_lane = a.q + (long long)(c0 + l0) * (G / 2) + t * (4 * W);
    const ST* s_warp = static_cast<const ST*>(a.scales) + c0 + l0;
    const ST* z_warp = static_cast<const ST*>(a.zeros) + c0 + l0;
    auto open_tile = [&]() {
      if (f_tile >= a.tiles) return;
      // rows past n read the last row again and are not stored
      // (n + 16 warps_n stays below 2^31: checked by the host)
      const uint32_t base = (uint32_t)((f_tile << a.warps_n_log) + wn) * 16u + g, end = (uint32_t)a.n - 1u;
      const uint64_t e0 = (uint64_t)min(base, end) * groups, e1 = (uint64_t)min(base + 8u, end) * groups;
      q0 = q_lane + e0 * (G / 2);
      q1 = q_lane + e1 * (G / 2);
      s0 = s_warp + e0;
      s1 = s_warp + e1;
      if constexpr (ZEROS) { z0 = z_warp + e0; z1 = z_warp + e1; }
      f_left = gk;
      f_tile += a.teams;
    };
    auto fetch = [&](int d) {
      if (f_left == 0) open_tile();
      if (f_left == 0) return;                       // nothing left (or no groups at all)
      --f_left;
      q4_load<W>(q0, w0[d]);
      q4_load<W>(q1, w1[d]);
      sc[d][0] = *s0++;
      sc[d][1] = *s1++;
      if constexpr (ZEROS) { zr[d][0] = *z0++; zr[d][1] = *z1++; }
      q0 += G / 2;
      q1 += G / 2;
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) fetch(d);        // weights fly while x is staged

    if (c0 != cta0) __syncthreads();                 // the last chunk's x has been used
    wild |= __syncthreads_or(q4_stage<XT, G, NT, PLANES, WARPS>(a, sm, c0, count));

    const bool first = c0 == cta0, last = c0 + count == cta1 && ksplit == 1;
#pragma unroll 1
    for (int tile = team, mine_at = 0; tile < a.tiles; tile += a.teams, ++mine_at) {
      float tot[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) tot[i][e] = 0.0f;
      uint32_t x_off = (uint32_t)(l0 * a.m) * 64u, g_off = (uint32_t)(l0 * a.m) * 8u;
#pragma unroll 1
      for (int left = gk; left > 0; left -= DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
          if (d >= left) break;
          float lo[NT][4], hi[NT][4];                // products with q 2^-24 and q 2^-20
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const uint32_t u0 = w0[d][w], u1 = w1[d][w], v0 = u0 >> 8, v1 = u1 >> 8;
            const uint32_t al0 = q4_pair<0, EXACT>(u0), al1 = q4_pair<0, EXACT>(u1);
            const uint32_t al2 = q4_pair<0, EXACT>(v0), al3 = q4_pair<0, EXACT>(v1);
            const uint32_t ah0 = q4_pair<4, EXACT>(u0), ah1 = q4_pair<4, EXACT>(u1);
            const uint32_t ah2 = q4_pair<4, EXACT>(v0), ah3 = q4_pair<4, EXACT>(v1);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              const uint32_t at = xa[i] ? xa[i] + x_off + w * x_word : zero_slot;
              if constexpr (PLANES == 1) {
                const uint4 b = q4_lds16(at);
                if (w == 0) {
                  q4_mma0(lo[i], al0, al1, al2, al3, b.x, b.y);
                  q4_mma0(hi[i], ah0, ah1, ah2, ah3, b.z, b.w);
                } else {
                  q4_mma(lo[i], al0, al1, al2, al3, b.x, b.y);
                  q4_mma(hi[i], ah0, ah1, ah2, ah3, b.z, b.w);
                }
              } else {
                // the tensor core cuts a sum off below its last bit: short
                // chains, smallest plane first, then rounded fp32 additions
                float l4[4], h4[4];
#pragma unroll
                for (int pl = PLANES - 1; pl >= 0; --pl) {
                  const uint4 b = q4_lds16(xa[i] ? at + (uint32_t)(pl * sm.plane) * 16u : at);
                  if (pl == PLANES - 1) {
                    q4_mma0(l4, al0, al1, al2, al3, b.x, b.y);
                    q4_mma0(h4, ah0, ah1, ah2, ah3, b.z, b.w);
                  } else {
                    q4_mma(l4, al0, al1, al2, al3, b.x, b.y);
                    q4_mma(h4, ah0, ah1, ah2, ah3, b.z, b.w);
                  }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  lo[i][e] = w == 0 ? l4[e] : lo[i][e] + l4[e];
                  hi[i][e] = w == 0 ? h4[e] : hi[i][e] + h4[e];
                }
              }
            }
          }
          constexpr float UNIT = EXACT ? 1.0f : 16777216.0f;         // 2^24
          const float f0 = to_f32(sc[d][0]) * UNIT, f1 = to_f32(sc[d][1]) * UNIT;
          float c0z = EXACT ? 0.0f : 8.0f, c1z = c0z;
          if constexpr (ZEROS) {
            c0z = to_f32(zr[d][0]) - (EXACT ? 8.0f : 0.0f);
            c1z = to_f32(zr[d][1]) - (EXACT ? 8.0f : 0.0f);
          }
          fetch(d);
#pragma unroll
          for (int i = 0; i < NT; ++i) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 gx = q4_lds8(ga[i][e] + g_off);     // (sum of x, scale)
              const float p0 = fmaf(hi[i][e], 0.0625f, lo[i][e]) * gx.y;
              const float p1 = fmaf(hi[i][e + 2], 0.0625f, lo[i][e + 2]) * gx.y;
              tot[i][e] = fmaf(f0, fmaf(-c0z, gx.x, p0), tot[i][e]);
              tot[i][e + 2] = fmaf(f1, fmaf(-c1z, gx.x, p1), tot[i][e + 2]);
            }
          }
          x_off += (uint32_t)a.m * 64u;
          g_off += (uint32_t)a.m * 8u;
        }
      }
      // the next tile starts in slot 0: turn the ring by what was used of it
#pragma unroll 1
      for (int r = gk % DEPTH; r > 0; --r) {
        uint32_t t0[W], t1[W];
        const ST ts0 = sc[0][0], ts1 = sc[0][1], tz0 = zr[0][0], tz1 = zr[0][1];
#pragma unroll
        for (int w = 0; w < W; ++w) { t0[w] = w0[0][w]; t1[w] = w1[0][w]; }
#pragma unroll
        for (int d = 0; d + 1 < DEPTH; ++d) {
#pragma unroll
          for (int w = 0; w < W; ++w) { w0[d][w] = w0[d + 1][w]; w1[d][w] = w1[d + 1][w]; }
          sc[d][0] = sc[d + 1][0]; sc[d][1] = sc[d + 1][1];
          zr[d][0] = zr[d + 1][0]; zr[d][1] = zr[d + 1][1];
        }
#pragma unroll
        for (int w = 0; w < W; ++w) { w0[DEPTH - 1][w] = t0[w]; w1[DEPTH - 1][w] = t1[w]; }
        sc[DEPTH - 1][0] = ts0; sc[DEPTH - 1][1] = ts1;
        zr[DEPTH - 1][0] = tz0; zr[DEPTH - 1][1] = tz1;
      }

      // the warps' partial sums of the tile meet in shared memory (one barrier
      // a tile: the other buffer is written before it, and this one is read
      // before the next tile's)
      float* buf = sm.red + (mine_at & 1) * (WARPS * RED);
      float* mine = buf + warp * RED;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = i * 8 + 2 * t + (e & 1);
          if (row < a.m) mine[row * 16 + g + (e >> 1) * 8] = tot[i][e];
        }
      }
      __syncthreads();
      int on = my_on, rest = my_rest;
#pragma unroll 1
      for (int i = threadIdx.x; i < per; i += WARPS * 32) {
        if (i != (int)threadIdx.x) { on = i / (16 * a.m); rest = i - on * (16 * a.m); }
        const float* part = buf + on * RED + rest;
        float y = first ? 0.0f : sm.sums[mine_at * per + i];
#pragma unroll 4
        for (int k = 0; k < warps_k; ++k) y += part[k * warps_n * RED];
        const long long col = ((long long)tile * warps_n + on) * 16 + rest % 16;
        if (!last) sm.sums[mine_at * per + i] = y;
        else if (col < a.n) static_cast<OT*>(a.out)[(rest / 16) * a.n + col] = from_f32<OT>(y);
      }
    }
  }

  if (ksplit > 1) {
    // the CTAs of the cluster share the outputs; each sums its share over all
    // ranks, in rank order
    q4_cluster_sync();
    const uint32_t local = static_cast<uint32_t>(__cvta_generic_to_shared(sm.sums));
    for (int tile = team, mine_at = 0; tile < a.tiles; tile += a.teams, ++mine_at) {
      for (int i = rank * WARPS * 32 + threadIdx.x; i < per; i += ksplit * WARPS * 32) {
        const int on = i / (16 * a.m), rest = i - on * (16 * a.m);
        float y = 0.0f;
        for (int c = 0; c < ksplit; ++c) {
          uint32_t base;
          float v;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(base) : "r"(local), "r"(c));
          asm volatile("ld.shared::cluster.f32 %0, [%1];"
                       : "=f"(v) : "r"(base + 4u * (uint32_t)(mine_at * per + i)));
          y += v;
        }
        const long long col = ((long long)tile * warps_n + on) * 16 + rest % 16;
        if (col < a.n) static_cast<OT*>(a.out)[(rest / 16) * a.n + col] = from_f32<OT>(y);
      }
    }
    q4_cluster_sync();                               // peers may still read this CTA's sums
  }
  if (wild) {
    __syncthreads();                                 // (the cluster's CTAs have stored as well)
    q4_wild_rows<XT, ST, OT, G, ZEROS, WARPS>(a, team);
  }
}

}  // namespace molten
