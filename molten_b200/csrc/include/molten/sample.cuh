// One token per row of logits from given random numbers:
//
//   w_i = e^((x_i - max x) / temperature); keep the top_k largest; of those the
//   fewest largest ones with weight >= top_p of theirs; of those the ones with
//   w >= min_p; the token is the first, by index, at which the running weight
//   of the kept exceeds u times their sum.  Equal logits count by index.
//
// Whether a token lies on this or that side of a border is the result, so
// weights and sums are held in 64 bits (with 2^17 kept tokens, fp32 weights
// would move one border in some hundred rows past its u), sums are taken in a
// fixed order, and every token kept is one of "x > tau, or x = tau and among
// the first `ties` of those": the two filters by rank become a value and a
// count.
//
// Bound by HBM (the logits, read once), for few rows by latency.  The CTAs of
// a cluster hold a row in shared memory as fp32, a run of consecutive tokens a
// thread (an odd number: no bank conflicts), and everything after the first
// pass stays on the SMs.  A threshold is found by narrowing an interval of
// values: 1024 bins of it are counted (integer atomics: their order changes
// nothing), the bins that can hold the border are selected, and when few
// enough tokens are left they are compared with one another directly.  For
// top_p a bin's weight is bounded by its edges' weights times its count; what
// lies above the remaining interval is summed exactly.  All CTAs of a cluster
// compute the same values from the same numbers, so they take the same steps.
//
// Weights: 2^(j / 256) from a table times a cubic (Taylor) in the rest of the
// exponent, |rest| <= ln 2 / 512: relative error below 2e-13, with 8 fp64
// operations where a library call takes some 30.
#pragma once

#include "molten/common.cuh"

namespace molten {

struct SampleArgs {
  const void* logits;              // [rows, vocab], rows row_stride elements apart
  const float* u;                  // [rows]
  const float* temperature;        // [rows], or null: the scalars below
  const int* top_k;
  const float* top_p;
  const float* min_p;
  int* out;                        // [rows]
  long long row_stride;
  int rows, vocab;
  int run;                         // tokens per thread
  int ranks;                       // CTAs of a cluster
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
};

constexpr int SAMPLE_THREADS = 256, SAMPLE_BINS = 1024, SAMPLE_LIST = 512;

struct SampleShared {
  double2 ex[2][8];                // exchanged values of the ranks
  double2 red[SAMPLE_THREADS / 32];
  double table[256];               // 2^(j / 256)
  unsigned hist[2][SAMPLE_BINS];
  float list[SAMPLE_LIST];         // this CTA's tokens of the last interval
  float all[SAMPLE_LIST];          // the cluster's
  unsigned long long wall[SAMPLE_LIST];
  int list_n, b0, b1, n0, n1;
};

__device__ __forceinline__ uint32_t sm_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint32_t sm_peer(const void* p, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(sm_addr(p)), "r"(rank));
  return r;
}

struct Sampler {
  const SampleArgs& a;
  SampleShared& s;
  float* xs;                       // this CTA's tokens: SAMPLE_THREADS runs
  int rank, tid, turn, hturn;
  float m;                         // largest logit
  double c, mc;                    // weights: 2^((x c + mc) / 256)

  __device__ __forceinline__ void sync() {
    if (a.ranks > 1)
      asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    else
      __syncthreads();
  }

  // Combine a pair of values of every thread of the cluster; the same result
  // everywhere (warps in order, then ranks in order).
  template <class F> __device__ __forceinline__ double2 combine(double2 v, F f) {
#pragma unroll
    for (int d = 16; d >= 1; d /= 2)
      v = f(v, make_double2(__shfl_xor_sync(0xffffffffu, v.x, d), __shfl_xor_sync(0xffffffffu, v.y, d)));
    if (tid % 32 == 0) s.red[tid / 32] = v;
    __syncthreads();
    v = s.red[0];
#pragma unroll
    for (int w = 1; w < SAMPLE_THREADS / 32; ++w) v = f(v, s.red[w]);
    if (a.ranks == 1) {
      __syncthreads();
      return v;
    }
    double2* ex = s.ex[turn & 1];                    // (two buffers: one barrier an exchange)
    ++turn;
    if (tid < a.ranks) {
      const uint32_t at = sm_peer(&ex[rank], tid);
      asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" :: "r"(at), "d"(v.x), "d"(v.y) : "memory");
    }
    sync();
    v = ex[0];
    for (int r = 1; r < a.ranks; ++r) v = f(v, ex[r]);
    return v;
  }
  __device__ __forceinline__ double2 sum2(double2 v) {
    return combine(v, [](double2 p, double2 q) { return make_double2(p.x + q.x, p.y + q.y); });
  }

  // Inclusive sums over the threads of the CTA; `all`: the CTA's total.
  __device__ __forceinline__ double2 scan2(double2 v, double2* all) {
    const int lane = tid % 32;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const double x = __shfl_up_sync(0xffffffffu, v.x, d), y = __shfl_up_sync(0xffffffffu, v.y, d);
      if (lane >= d) { v.x += x; v.y += y; }
    }
    if (lane == 31) s.red[tid / 32] = v;
    __syncthreads();
    double2 before = make_double2(0.0, 0.0), total = before;
#pragma unroll
    for (int w = 0; w < SAMPLE_THREADS / 32; ++w) {
      if (w == tid / 32) before = total;
      total.x += s.red[w].x;
      total.y += s.red[w].y;
    }
    __syncthreads();
    *all = total;
    return make_double2(v.x + before.x, v.y + before.y);
  }

  // 2^(t / 256), t <= 0
  __device__ __forceinline__ double power(double t) const {
    if (!(t > -256.0 * 1000.0)) return 0.0;          // below 2^-1000, -inf, NaN
    const double big = t + 6755399441055744.0;       // 1.5 2^52: round(t) in the low bits
    const int k = __double2loint(big);
    const double r = t - (big - 6755399441055744.0);
    const double k1 = 0.0027076061740622863;         // ln 2 / 256
    const double p = fma(r, fma(r, fma(r, k1 * k1 * k1 / 6.0, k1 * k1 / 2.0), k1), 1.0);
    const double w = s.table[k & 255] * p;
    return __hiloint2double(__double2hiint(w) + ((k >> 8) << 20), __double2loint(w));
  }
  __device__ __forceinline__ double weight(float x) const {
    return x == m ? 1.0 : power(fma((double)x, c, mc));
  }

  // The border in [lo, hi], among tokens x >= lo.  WEIGHT = false: the token
  // of rank `goal` (from 1) counted from the largest; n is the number above
  // hi.  WEIGHT = true: the first token at which the running weight reaches
  // `goal`; n is the weight above hi.  Returns its value; *ties: how many
  // tokens of that value belong to the kept.
  template <bool WEIGHT>
  __device__ __forceinline__ float border(float lo, float hi, double n, double goal, double* ties) {
#pragma unroll 1
    for (int step = 0; step < 64; ++step) {
      if (!(lo < hi)) {
        *ties = WEIGHT ? ceil((goal - n) / weight(hi)) : goal - n;
        return hi;
      }
      // (halves: the difference of two finite values stays finite)
      const float span = 0.5f * hi - 0.5f * lo;
      const float inv = fminf((float)(SAMPLE_BINS - 1) / span, 3.0e38f);
      auto bin = [&](float x) { return min(SAMPLE_BINS - 1, (int)((0.5f * hi - 0.5f * x) * inv)); };
      unsigned* hist = s.hist[hturn & 1];
      ++hturn;
      for (int b = tid; b < SAMPLE_BINS; b += SAMPLE_THREADS) hist[b] = 0u;
      if (tid == 0) { s.b0 = SAMPLE_BINS - 1; s.b1 = SAMPLE_BINS - 1; s.list_n = 0; }
      __syncthreads();
      const float* mine = xs + tid * a.run;
#pragma unroll 4
      for (int i = 0; i < a.run; ++i) {
        const float x = mine[i];
        if (x >= lo && x <= hi) atomicAdd(&hist[bin(x)], 1u);
      }
      sync();
      constexpr int PER = SAMPLE_BINS / SAMPLE_THREADS;
      uint4 cnt = make_uint4(0u, 0u, 0u, 0u);        // bins 4 tid .. 4 tid + 3 of the cluster
      static_assert(PER == 4, "a thread's bins are one 16-byte load");
      for (int r = 0; r < a.ranks; ++r) {
        uint4 v;
        if (a.ranks == 1) {
          v = *reinterpret_cast<const uint4*>(&hist[4 * tid]);
        } else {
          asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(sm_peer(&hist[4 * tid], r)));
        }
        cnt.x += v.x; cnt.y += v.y; cnt.z += v.z; cnt.w += v.w;
      }
      const unsigned cs[4] = {cnt.x, cnt.y, cnt.z, cnt.w};
      // counts before the thread's bins, and the bounds of the weight up to each
      double2 all, at;
      at = scan2(make_double2((double)(cs[0] + cs[1] + cs[2] + cs[3]), 0.0), &all);
      const double count0 = at.x - (double)(cs[0] + cs[1] + cs[2] + cs[3]);
      if constexpr (WEIGHT) {
        // a token of bin b is above the bin's lower edge and not above its
        // upper one; 0.01 bins cover the fp32 rounding of the bin's number
        double up[4], least_of[4];
        const double width = 2.0 / (double)inv;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int b = 4 * tid + q;
          const double high = fmin((double)m, (double)hi - ((double)b - 0.01) * width);
          // (the last bin also holds everything down to lo)
          const double low = b == SAMPLE_BINS - 1 ? (double)lo : (double)hi - ((double)b + 1.01) * width;
          up[q] = power(high * c + mc) * (1.0 + 1e-11);
          least_of[q] = power(low * c + mc) * (1.0 - 1e-11);
        }
        double2 part[4], run = make_double2(0.0, 0.0);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          run.x += (double)cs[q] * up[q];
          run.y += (double)cs[q] * least_of[q];
          part[q] = run;
        }
        const double2 incl = scan2(run, &all);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const double most = n + (incl.x - run.x) + part[q].x, least = n + (incl.y - run.y) + part[q].y;
          if (most * (1.0 + 1e-12) >= goal) atomicMin(&s.b0, 4 * tid + q);
          if (least * (1.0 - 1e-12) >= goal) atomicMin(&s.b1, 4 * tid + q);
        }
      } else {
        double before = count0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const double up = before + (double)cs[q];
          if (n + up >= goal) { atomicMin(&s.b0, 4 * tid + q); atomicMin(&s.b1, 4 * tid + q); }
          before = up;
        }
      }
      __syncthreads();
      const int b0 = s.b0, b1 = max(s.b1, s.b0);
      {
        double before = count0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const double up = before + (double)cs[q];
          if (4 * tid + q == b0) s.n0 = (int)before;
          if (4 * tid + q == b1) s.n1 = (int)up;
          before = up;
        }
      }
      __syncthreads();
      const int left = s.n1 - s.n0;                  // tokens of bins b0 .. b1
      const bool listed = left <= SAMPLE_LIST;
      // what lies above, exactly; the interval's own extremes, or its tokens
      double above = 0.0;
      float top = -INFINITY, low = INFINITY;
#pragma unroll 1
      for (int i = 0; i < a.run; ++i) {
        const float x = mine[i];
        if (!(x >= lo && x <= hi)) continue;
        const int b = bin(x);
        if (b < b0) {
          above += WEIGHT ? weight(x) : 1.0;
        } else if (b <= b1) {
          top = fmaxf(top, x);
          low = fminf(low, x);
          if (listed) s.list[atomicAdd(&s.list_n, 1)] = x;
        }
      }
      const double2 ext = combine(make_double2((double)top, -(double)low), [](double2 p, double2 q) {
        return make_double2(fmax(p.x, q.x), fmax(p.y, q.y)); });
      n += sum2(make_double2(above, 0.0)).x;
      hi = (float)ext.x;
      lo = (float)-ext.y;
      if (!listed || !(lo < hi)) continue;

      // few are left: gather them and compare each with all others.  Weights
      // as integers of 2^-52, so that the order of the list changes nothing.
      if (a.ranks > 1) sync();                       // every rank's list is complete
      int at0 = 0;
      for (int r = 0; r < a.ranks; ++r) {
        int have;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(have) : "r"(sm_peer(&s.list_n, r)));
        for (int i = tid; i < have; i += SAMPLE_THREADS) {
          float x;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(sm_peer(&s.list[i], r)));
          s.all[at0 + i] = x;
          s.wall[at0 + i] = WEIGHT ? (unsigned long long)__double2ll_rn(weight(x) * 4503599627370496.0) : 1ull;
        }
        at0 += have;
      }
      sync();                                        // (peers have read this CTA's list)
      const double unit = WEIGHT ? 4503599627370496.0 : 1.0;
      const double need = (goal - n) * unit;         // weight that the listed have to bring
      float best = -INFINITY;
      unsigned long long best_above = 0ull;
      for (int i = tid; i < left; i += SAMPLE_THREADS) {
        const float x = s.all[i];
        unsigned long long gt = 0ull, ge = 0ull;
#pragma unroll 4
        for (int j = 0; j < left; ++j) {
          const unsigned long long w = s.wall[j];
          const float y = s.all[j];
          if (y > x) gt += w;
          if (y >= x) ge += w;
        }
        // the largest value whose running weight reaches the goal
        if ((double)ge >= need && x > best) { best = x; best_above = gt; }
      }
      const double2 win = combine(make_double2((double)best, 0.0), [](double2 p, double2 q) {
        return make_double2(fmax(p.x, q.x), 0.0); });
      const float tau = win.x == -INFINITY ? lo : (float)win.x;
      // its tokens above, the same number wherever it is found
      if (best == tau) s.wall[0] = best_above;       // (every writer writes the same)
      __syncthreads();
      const double gt = win.x == -INFINITY ? 0.0 : (double)s.wall[0];
      const double w = WEIGHT ? weight(tau) * unit : 1.0;
      *ties = win.x == -INFINITY ? 1e18 : ceil((need - gt) / w);
      __syncthreads();
      return tau;
    }
    *ties = 1e18;
    return lo;
  }
};

template <typename T>
__device__ __forceinline__ void sample_row(const SampleArgs& a, uint8_t* raw) {
  SampleShared& sh = *reinterpret_cast<SampleShared*>(raw);
  float* xs = reinterpret_cast<float*>(raw + sizeof(SampleShared));
  const int rank = blockIdx.x % a.ranks, row = blockIdx.x / a.ranks, tid = threadIdx.x;
  Sampler k{a, sh, xs, rank, tid, 0, 0, 0.0f, 0.0, 0.0};
  const int part = SAMPLE_THREADS * a.run, base = rank * part;
  const int n = max(0, min(part, a.vocab - base));
  const T* src = static_cast<const T*>(a.logits) + row * a.row_stride + base;
  const float u = a.u[row];
  const float temperature = a.temperature ? a.temperature[row] : a.temperature_all;
  const int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all;
  const float min_p = a.min_p ? a.min_p[row] : a.min_p_all;

  // the tokens of this CTA; NaN as -inf, +inf as the largest finite value
  float top = -INFINITY, low = INFINITY;
  int finite = 0;
  auto take = [&](int i, float x) {
    x = x != x ? -INFINITY : fminf(x, 3.402823466e38f);
    xs[i] = x;
    top = fmaxf(top, x);
    if (x != -INFINITY) { low = fminf(low, x); ++finite; }
  };
  if constexpr (sizeof(T) == 2) {
    const int head = n > 0 && (reinterpret_cast<uintptr_t>(src) & 2) ? 1 : 0;
    if (head && tid == 0) take(0, to_f32(src[0]));
    const int pairs = (n - head) / 2;
    const uint32_t* src2 = reinterpret_cast<const uint32_t*>(src + head);
#pragma unroll 8
    for (int i = tid; i < pairs; i += SAMPLE_THREADS) {
      const uint32_t v = __ldg(src2 + i);
      const Slot<T, 2> two = *reinterpret_cast<const Slot<T, 2>*>(&v);
      take(head + 2 * i, to_f32(two.v[0]));
      take(head + 2 * i + 1, to_f32(two.v[1]));
    }
    const int done = head + 2 * pairs;
    if (done < n && tid == 0) take(done, to_f32(src[done]));
  } else {
#pragma unroll 8
    for (int i = tid; i < n; i += SAMPLE_THREADS) take(i, __ldg(src + i));
  }
  for (int i = n + tid; i < part; i += SAMPLE_THREADS) xs[i] = -INFINITY;
  sh.table[tid] = exp2((double)tid * (1.0 / 256.0));
  const double2 ext = k.combine(make_double2((double)top, -(double)low), [](double2 p, double2 q) {
    return make_double2(fmax(p.x, q.x), fmax(p.y, q.y)); });
  k.m = (float)ext.x;
  const float least = (float)-ext.y;
  const float* mine = xs + tid * a.run;
  const int first = base + tid * a.run;              // index of the thread's first token

  if (k.m == -INFINITY) {                            // nothing can be drawn
    if (rank == 0 && tid == 0) a.out[row] = -1;
    if (a.ranks > 1) k.sync();
    return;
  }
  if (!(temperature > 0.0f)) {
    double at = 2147483647.0;
    for (int i = 0; i < a.run; ++i)
      if (mine[i] == k.m) { at = (double)(first + i); break; }
    const double2 best = k.combine(make_double2(-at, 0.0), [](double2 p, double2 q) {
      return make_double2(fmax(p.x, q.x), 0.0); });
    if (rank == 0 && tid == 0) a.out[row] = (int)-best.x;
    return;
  }
  k.c = 256.0 * 1.4426950408889634074 / (double)temperature;
  k.mc = -(double)k.m * k.c;

  // kept: x > tau, and the first `ties` of x = tau
  float tau = -INFINITY;
  double ties = 0.0;
  if (top_k > 0 && top_k < a.vocab) {
    const double have = k.sum2(make_double2((double)finite, 0.0)).x;
    if ((double)top_k < have) tau = k.border<false>(least, k.m, 0.0, (double)top_k, &ties);
  }
  if (top_p < 1.0f) {
    double w = 0.0;
    float lowest = INFINITY;
#pragma unroll 4
    for (int i = 0; i < a.run; ++i) {
      const float x = mine[i];
      if (x > tau) { w += k.weight(x); lowest = fminf(lowest, x); }
    }
    const double2 got = k.combine(make_double2(w, -(double)lowest), [](double2 p, double2 q) {
      return make_double2(p.x + q.x, fmax(p.y, q.y)); });
    const double wt = tau == -INFINITY ? 0.0 : k.weight(tau);
    const double goal = fmax((double)top_p, 0.0) * (got.x + ties * wt);
    if (goal > got.x) {                              // inside the ties of top_k's border
      ties = fmin(ties, fmax(1.0, ceil((goal - got.x) / wt)));
    } else if (goal > 0.0) {
      // start where the weights matter: below m - 40 T they are under 5e-18
      const float near = (float)fmax(-got.y, (double)k.m - 40.0 * (double)temperature);
      double above = 0.0;
      float start = fmaxf((float)-got.y, near);
      tau = k.border<true>(start, k.m, above, goal, &ties);
      ties = fmax(ties, 1.0);
    } else {
      tau = k.m;                                     // the largest token at least
      ties = 1.0;
    }
  }

  // the kept tokens' weights per thread; ties in index order
  const double floor_w = fmin((double)min_p, 1.0);   // the largest token is always kept
  const bool has_floor = min_p > 0.0f;
  double w = 0.0, eq = 0.0;
#pragma unroll 4
  for (int i = 0; i < a.run; ++i) {
    const float x = mine[i];
    if (x > tau) {
      const double v = k.weight(x);
      if (!has_floor || v >= floor_w) w += v;
    }
    eq += x == tau ? 1.0 : 0.0;
  }
  if (tau == -INFINITY) eq = 0.0;
  const double wt = tau == -INFINITY ? 0.0 : k.weight(tau);
  if (has_floor && wt < floor_w) ties = 0.0;
  double2 all;
  // ties before the thread's run
  double2 inc = k.scan2(make_double2(eq, 0.0), &all);
  auto ranks_before = [&](double mine_total, double* total) {
    // this rank's predecessors' sum and the sum of all, in rank order
    double before = 0.0;
    *total = mine_total;
    if (a.ranks > 1) {
      double2* ex = sh.ex[k.turn & 1];
      ++k.turn;
      if (tid < a.ranks) {
        const uint32_t to = sm_peer(&ex[rank], tid);
        asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" :: "r"(to), "d"(mine_total), "d"(0.0) : "memory");
      }
      k.sync();
      double t = 0.0;
      for (int r = 0; r < a.ranks; ++r) {
        if (r == rank) before = t;
        t += ex[r].x;
      }
      *total = t;
    }
    return before;
  };
  double total;
  const double eq0 = ranks_before(all.x, &total) + inc.x - eq;
  const double in = fmin(fmax(ties - eq0, 0.0), eq);  // ties of this run that are kept
  const double sum = w + in * wt;
  inc = k.scan2(make_double2(sum, 0.0), &all);
  const double before = ranks_before(all.x, &total);
  const double goal = (u > 0.0f ? (double)fminf(u, 0.99999994f) : 0.0) * total;
  // the first thread of the row whose running weight exceeds the goal
  const double upto = before + inc.x;
  const double own = sum > 0.0 && upto > goal ? (double)(rank * SAMPLE_THREADS + tid) : 1e9;
  const double2 who = k.combine(make_double2(-own, 0.0), [](double2 p, double2 q) {
    return make_double2(fmax(p.x, q.x), 0.0); });
  const int owner = (int)-who.x;
  if (owner / SAMPLE_THREADS != rank || owner % SAMPLE_THREADS / 32 != tid / 32) return;
  // its warp looks through its run, 32 tokens at a time
  const int lane = tid % 32, src_lane = owner % 32;
  double run = __shfl_sync(0xffffffffu, upto - sum, src_lane);
  double seen_eq = __shfl_sync(0xffffffffu, eq0, src_lane);
  const float* runx = xs + (owner % SAMPLE_THREADS) * a.run;
  int found = -1, last = 0;
  for (int i0 = 0; i0 < a.run && found < 0; i0 += 32) {
    const float x = i0 + lane < a.run ? runx[i0 + lane] : -INFINITY;
    const bool tie = x == tau && x != -INFINITY;
    const unsigned tied = __ballot_sync(0xffffffffu, tie);
    const double mine_eq = seen_eq + (double)__popc(tied & ((1u << lane) - 1u));
    double v = 0.0;
    if (x > tau) {
      v = k.weight(x);
      if (has_floor && v < floor_w) v = 0.0;
    } else if (tie && mine_eq < ties) {
      v = wt;
    }
    const unsigned kept = __ballot_sync(0xffffffffu, v > 0.0);
    double acc = v;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const double y = __shfl_up_sync(0xffffffffu, acc, d);
      if (lane >= d) acc += y;
    }
    const unsigned over = __ballot_sync(0xffffffffu, v > 0.0 && run + acc > goal);
    if (over) found = i0 + __ffs(over) - 1;
    if (kept) last = i0 + 31 - __clz(kept);
    run += __shfl_sync(0xffffffffu, acc, 31);
    seen_eq += (double)__popc(tied);
  }
  if (lane == 0)
    a.out[row] = rank * part + (owner % SAMPLE_THREADS) * a.run + (found >= 0 ? found : last);
}

}  // namespace molten
