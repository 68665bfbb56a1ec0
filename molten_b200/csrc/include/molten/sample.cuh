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
// The logits are read once; what bounds it is the work behind that: some 100
// instructions a token, and for few rows the latency of the steps.  The CTAs of
// a cluster hold a row in shared memory in its own type, a run of consecutive
// tokens a thread (an odd number of 32-bit words: no bank conflicts), and
// everything after the first pass stays on the SMs.  What the filters can keep
// is found by counting the tokens in 1024 bins of values (integer atomics:
// their order changes nothing) and bounding a bin's weight by its edges'
// weights times its count; those tokens are packed together, in order of their
// index, and the rest works on them alone, every lane at work: exact weights,
// the borders, the draw.  (With the weights computed where the tokens lay,
// behind a branch that some lane of a warp took nearly always, that pass took
// 52000 cycles; packed, under 10000.)  Few packed tokens go to the first CTA,
// which finishes without the cluster's barriers.  A border is found by narrowing
// an interval of values, bin by bin, until few enough tokens are left to compare
// each with all.  Rows whose kept tokens do not fit the packed list go the same
// way with the whole row in its place.
//
// Measured: 1 x 32768 fp32 with top_k and top_p 22.0 us; 64 x 131072 bf16 with
// top_p and min_p, 16000 tokens kept, 108 us (before the dropped ones' 64-bit
// weights 100; 132 with the tokens that are surely kept left in the border's
// search, 109 with their weights behind a branch); 256 x 100003 fp32, some rows
// with each filter, 157 us; the same unfiltered 103 us (0.99 TB/s).
//
// The tail that top_p surely drops, of which it needs nothing but the total, has
// 64-bit terms as well: with ex2.approx ones the total of thousands was off by near
// 1e-8 of itself, which moved the border past a token for one row in 10^3.
//
// All CTAs of a cluster compute the same values from the same numbers, so they
// take the same steps.
//
// Weights: 2^(j / 256) from a table times a cubic (Taylor) in the rest of the
// exponent, |rest| <= ln 2 / 512: relative error below 2e-13, with 9 fp64
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
  int run;                         // tokens per thread: an odd number of 32-bit words
  int ranks;                       // CTAs of a cluster
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
};

constexpr int SAMPLE_BINS = 1024, SAMPLE_LIST = 512, SAMPLE_MAX_RANKS = 8;

struct SampleShare { float x, y; double z, w; };     // two maxima and two sums of a warp or rank
struct SampleSums { double x; float y, z; };         // sums of a thread

template <typename T, int THREADS>
struct SampleShared {
  static constexpr int PACKED = THREADS * 32 / (int)sizeof(T);
  SampleShare ex[2][SAMPLE_MAX_RANKS];   // exchanged values of the ranks
  SampleShare red[32];
  double table[256];               // 2^(j / 256)
  union {                          // (a cluster barrier lies between their uses)
    unsigned hist[SAMPLE_BINS];
    unsigned long long wall[SAMPLE_LIST];          // weights of `all`
  };
  float list[SAMPLE_LIST];         // this CTA's tokens of the last interval
  float all[SAMPLE_LIST];          // the cluster's
  T packed[PACKED];                // what the filters can keep, by index
  unsigned short packed_at[PACKED];         // index within its CTA's part
  int starts[SAMPLE_MAX_RANKS];    // the ranks' first places, of all that is packed
  int list_n, b0, b1, n0, n1, turn, pad[2];
};

__device__ __forceinline__ uint32_t sm_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint32_t sm_peer(const void* p, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(sm_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void sm_sync(int ranks) {
  if (ranks > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else
    __syncthreads();
}

template <typename E>
__device__ __forceinline__ void sm_put(uint32_t base, int i, E v) {
  if constexpr (sizeof(E) == 2)
    asm volatile("st.shared::cluster.u16 [%0], %1;" :: "r"(base + 2u * i), "h"(*reinterpret_cast<unsigned short*>(&v)) : "memory");
  else
    asm volatile("st.shared::cluster.f32 [%0], %1;" :: "r"(base + 4u * i), "f"(v) : "memory");
}

// Every rank's share in ex[0 .. ranks): published by each, one barrier.  (Two
// buffers in turn: what the last exchange left may still be read.)
template <class S>
__device__ __forceinline__ const SampleShare* sm_publish(S& s, int ranks, int rank, const SampleShare& v) {
  SampleShare* ex = s.ex[s.turn & 1];
  if (ranks > 1) {
    if ((int)threadIdx.x < ranks) {
      const uint32_t at = sm_peer(&ex[rank], threadIdx.x);
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" :: "r"(at), "f"(v.x), "f"(v.y) : "memory");
      asm volatile("st.shared::cluster.f64 [%0], %1;" :: "r"(at + 8u), "d"(v.z) : "memory");
      asm volatile("st.shared::cluster.f64 [%0], %1;" :: "r"(at + 16u), "d"(v.w) : "memory");
    }
  } else if (threadIdx.x == 0) {
    ex[0] = v;
  }
  sm_sync(ranks);
  if (threadIdx.x == 0) ++s.turn;                    // (read again only behind the next barrier)
  return ex;
}

// The code below is kept small: a CTA runs most of it once, and with loops
// unrolled (130 KB in all) its time went on fetching instructions.

// Maxima and sums over the first 2 `half` lanes, the same in each of them.
__device__ __forceinline__ void sm_lanes(SampleShare& v, int half) {
#pragma unroll 1
  for (int d = half; d >= 1; d /= 2) {
    v.x = fmaxf(v.x, __shfl_xor_sync(0xffffffffu, v.x, d));
    v.y = fmaxf(v.y, __shfl_xor_sync(0xffffffffu, v.y, d));
    v.z += __shfl_xor_sync(0xffffffffu, v.z, d);
    v.w += __shfl_xor_sync(0xffffffffu, v.w, d);
  }
}

// Maxima of x and y and the sums of z and w over every thread of the cluster, the
// same result everywhere.
template <int THREADS, class S>
__device__ __noinline__ SampleShare sm_combine(S& s, int ranks, int rank, SampleShare v) {
  const int lane = threadIdx.x % 32;
  sm_lanes(v, 16);
  if (lane == 0) s.red[threadIdx.x / 32] = v;
  __syncthreads();
  if (threadIdx.x < 32) {                            // (what the publishing threads need)
    v = s.red[lane % (THREADS / 32)];
    sm_lanes(v, THREADS / 64);
  }
  const SampleShare* ex = sm_publish(s, ranks, rank, v);
  v = ex[lane & (ranks - 1)];                        // (a power of two)
  sm_lanes(v, ranks / 2);
  return v;
}

// Inclusive sums over the threads of the CTA; *all: its totals.
template <int THREADS, class S>
__device__ __noinline__ SampleSums sm_scan(S& s, SampleSums v, SampleSums* all) {
  constexpr int WARPS = THREADS / 32;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  SampleSums* red = reinterpret_cast<SampleSums*>(s.red);
  SampleSums own = v;
#pragma unroll 1
  for (int turn = 0; turn < 2; ++turn) {             // the warp's lanes, then the warps
#pragma unroll 1
    for (int d = 1; d < 32; d *= 2) {
      const double x = __shfl_up_sync(0xffffffffu, v.x, d);
      const float y = __shfl_up_sync(0xffffffffu, v.y, d), z = __shfl_up_sync(0xffffffffu, v.z, d);
      if (lane >= d) { v.x += x; v.y += y; v.z += z; }
    }
    if (turn == 1) break;
    own = v;
    if (lane == 31) red[warp] = v;
    __syncthreads();
    v = lane < WARPS ? red[lane] : SampleSums{0.0, 0.0f, 0.0f};
  }
  __syncthreads();
  *all = {__shfl_sync(0xffffffffu, v.x, 31), __shfl_sync(0xffffffffu, v.y, 31), __shfl_sync(0xffffffffu, v.z, 31)};
  const int prev = max(warp - 1, 0);
  const double x = __shfl_sync(0xffffffffu, v.x, prev);
  const float y = __shfl_sync(0xffffffffu, v.y, prev), z = __shfl_sync(0xffffffffu, v.z, prev);
  if (warp > 0) { own.x += x; own.y += y; own.z += z; }
  return own;
}

// f(i, x) for every token of a thread's run, in order.
template <int UNROLL = 8, typename T, class F>
__device__ __forceinline__ void sm_each(const T* mine, int run, F f) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t* words = reinterpret_cast<const uint32_t*>(mine);
#pragma unroll UNROLL / 2
    for (int i = 0; i < run; i += 2) {
      const uint32_t v = words[i / 2];
      const Slot<T, 2> two = *reinterpret_cast<const Slot<T, 2>*>(&v);
      f(i, to_f32(two.v[0]));
      f(i + 1, to_f32(two.v[1]));
    }
  } else {
#pragma unroll UNROLL
    for (int i = 0; i < run; ++i) f(i, mine[i]);
  }
}

// f(i, x) for the few tokens of a run with want(x).  The comparisons of 8 tokens
// are made without branches, and a thread turns to f where one held.
template <typename T, class W, class F>
__device__ __forceinline__ void sm_few(const T* mine, int run, W want, F f) {
  constexpr int STEP = 8;
  int i = 0;
#pragma unroll 1
  for (; i + STEP <= run; i += STEP) {
    unsigned hits = 0u;
    if constexpr (sizeof(T) == 2) {
      const uint32_t* words = reinterpret_cast<const uint32_t*>(mine + i);
#pragma unroll
      for (int j = 0; j < STEP / 2; ++j) {
        const uint32_t v = words[j];
        const Slot<T, 2> two = *reinterpret_cast<const Slot<T, 2>*>(&v);
        hits |= (want(to_f32(two.v[0])) ? 1u : 0u) << (2 * j);
        hits |= (want(to_f32(two.v[1])) ? 1u : 0u) << (2 * j + 1);
      }
    } else {
#pragma unroll
      for (int j = 0; j < STEP; ++j) hits |= (want(to_f32(mine[i + j])) ? 1u : 0u) << j;
    }
    while (hits) {
      const int j = __ffs(hits) - 1;
      hits &= hits - 1u;
      f(i + j, to_f32(mine[i + j]));
    }
  }
#pragma unroll 1
  for (; i < run; ++i)
    if (want(to_f32(mine[i]))) f(i, to_f32(mine[i]));
}

// The bins of an interval of values, from the largest down.
struct SampleBins {
  static constexpr int BINS = SAMPLE_BINS;
  float hi, inv;
  __device__ __forceinline__ SampleBins(float lo, float hi_) : hi(hi_) {
    // (halves: the difference of two finite values stays finite)
    inv = fminf((float)(BINS - 1) / (0.5f * hi - 0.5f * lo), 3.0e38f);
  }
  // rounded to the nearest by an addition (the conversion to an integer runs at
  // an eighth of its rate): bin b holds [b - 1/2, b + 1/2]
  __device__ __forceinline__ int of(float x) const {
    return __float_as_int(fminf((0.5f * hi - 0.5f * x) * inv, (float)(BINS - 1)) + 12582912.0f) & 0xffff;
  }
};

template <typename T, int THREADS>
struct Sampler {
  static constexpr int BINS = SAMPLE_BINS, PER = BINS / THREADS;         // bins, and of a thread
  typedef SampleBins Bins;
  SampleShared<T, THREADS>& s;
  const T* mine;                   // this thread's run
  int run, ranks, rank, tid;
  float m, cut;                    // largest logit; below this one weights are 0
  double c;                        // weights: 2^((x - m) c / 256)
  float sure;                      // top_p keeps all above this one (no top_k)

  // 2^(t / 256), -256000 <= t <= 0 (the cut's is at least -254900)
  __device__ __forceinline__ double power(double t) const {
    const double big = t + 6755399441055744.0;       // 1.5 2^52: round(t) in the low bits
    const int k = __double2loint(big);
    const double r = t - (big - 6755399441055744.0);
    const double k1 = 0.0027076061740622863;         // ln 2 / 256
    const double p = fma(r, fma(r, fma(r, k1 * k1 * k1 / 6.0, k1 * k1 / 2.0), k1), 1.0);
    const double w = s.table[k & 255] * p;
    return __hiloint2double(__double2hiint(w) + ((k >> 8) << 20), __double2loint(w));
  }
  // (no branch: what the cut leaves out is computed at the cut and dropped)
  __device__ __forceinline__ double weight(float x) const {
    const double w = power(((double)fmaxf(x, cut) - (double)m) * c);
    return x >= cut ? w : 0.0;
  }

  // Counters for the bins of the next interval, zero behind the barrier.
  __device__ __forceinline__ void open_bins() {
#pragma unroll
    for (int q = 0; q < PER; ++q) s.hist[q * THREADS + tid] = 0u;
    if (tid == 0) { s.b0 = BINS - 1; s.b1 = BINS - 1; s.list_n = 0; }
    __syncthreads();
  }
  // The counts of this thread's bins (PER tid and on) in the whole cluster
  // (behind a cluster barrier).
  __device__ __forceinline__ void merge_bins(unsigned (&cs)[PER]) {
    static_assert(PER == 4 || PER == 2, "a thread's bins are one load");
    uint4 got[SAMPLE_MAX_RANKS];
#pragma unroll
    for (int r = 0; r < SAMPLE_MAX_RANKS; ++r) {
      got[r] = make_uint4(0u, 0u, 0u, 0u);
      if (r >= ranks) continue;
      const uint32_t at = sm_peer(&s.hist[PER * tid], r);
      if constexpr (PER == 4)
        asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(got[r].x), "=r"(got[r].y), "=r"(got[r].z), "=r"(got[r].w) : "r"(at));
      else
        asm volatile("ld.shared::cluster.v2.u32 {%0,%1}, [%2];" : "=r"(got[r].x), "=r"(got[r].y) : "r"(at));
    }
    uint4 sum = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int r = 0; r < SAMPLE_MAX_RANKS; ++r) {
      sum.x += got[r].x; sum.y += got[r].y; sum.z += got[r].z; sum.w += got[r].w;
    }
    cs[0] = sum.x; cs[1] = sum.y;
    if constexpr (PER == 4) { cs[2] = sum.z; cs[3] = sum.w; }
  }
  // The selected bins b0 .. b1 (chosen with atomicMin) and their tokens.
  __device__ __forceinline__ int close_bins(int before, const unsigned (&cs)[PER], int* b0, int* b1) {
    __syncthreads();
    *b0 = s.b0;
    *b1 = max(s.b1, *b0);
    int upto = before;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      if (PER * tid + q == *b0) s.n0 = upto;
      upto += (int)cs[q];
      if (PER * tid + q == *b1) s.n1 = upto;
    }
    __syncthreads();
    return s.n1 - s.n0;
  }

  // Count the tokens of `hist` bins over the cluster and select the bins that
  // can hold a border.  by_weight = false: the bin of the token of rank `goal`.
  // by_weight = true: those that can hold the first token at which n and the
  // running weight reach the goal; goal < 0: `share` of all that is counted.
  // Returns the selected bins' tokens.
  __device__ __noinline__ int select_bins(bool by_weight, const Bins& bins, float lo, double n, double goal, double share, int* b0, int* b1) {
    sm_sync(ranks);
    unsigned cs[PER];
    merge_bins(cs);
    // a token of bin b is above the bin's lower edge and not above its upper
    // one.  Bounds in fp32: 0.01 bins cover the rounding of the bin's number,
    // 3e-5 that of exponents (up to 58, a few 2^-24 of that), of ex2.approx
    // (2^-22) and of the sums
    // (half differences, as in SampleBins: two finite values may lie further apart
    // than the largest one)
    const float width = 1.0f / bins.inv, c1 = (float)c * (1.0f / 128.0f), gap = 0.5f * bins.hi - 0.5f * m;
    float most[PER], least[PER];
    SampleSums own = {0.0, 0.0f, 0.0f};              // tokens, the most and the least weight
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int b = PER * tid + q;
      own.x += (double)cs[q];
      if (by_weight) {
        const float high = fminf(0.0f, gap - ((float)b - 0.51f) * width);
        // (the last bin also holds everything down to lo)
        const float low = b == BINS - 1 ? 0.5f * lo - 0.5f * m : gap - ((float)b + 0.51f) * width;
        own.y += (float)cs[q] * fast_exp2(high * c1);
        own.z += (float)cs[q] * fast_exp2(low * c1);
      }
      most[q] = own.y;
      least[q] = own.z;
    }
    SampleSums all;
    const SampleSums incl = sm_scan<THREADS>(s, own, &all);
    const int before = (int)(incl.x - own.x);
    if (by_weight) {
      const float wide_up = 1.00003f, wide_down = 0.99997f;
      const double goal0 = goal >= 0.0 ? goal : share * (double)(all.z * wide_down);
      const double goal1 = goal >= 0.0 ? goal : share * (double)(all.y * wide_up);
#pragma unroll
      for (int q = PER - 1; q >= 0; --q) {
        if (n + (double)(((incl.y - own.y) + most[q]) * wide_up) >= goal0) atomicMin(&s.b0, PER * tid + q);
        if (n + (double)(((incl.z - own.z) + least[q]) * wide_down) >= goal1) atomicMin(&s.b1, PER * tid + q);
      }
    } else {
      int upto = before;
      const int want = (int)goal;
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        if (upto < want && want <= upto + (int)cs[q]) { s.b0 = PER * tid + q; s.b1 = PER * tid + q; }
        upto += (int)cs[q];
      }
    }
    return close_bins(before, cs, b0, b1);
  }

  // The listed tokens of every rank, compared with one another: the largest
  // value at which the weight from the top (by_weight; else the count) reaches
  // `need`.  -inf: none does.  *ties: how many of its tokens that takes.
  // Weights as integers of 2^-52, so that the order of the list changes
  // nothing.
  __device__ __noinline__ float pick(bool by_weight, double need, double* ties) {
    const double unit = by_weight ? 4503599627370496.0 : 1.0;
    int part[SAMPLE_MAX_RANKS], have = 0;
#pragma unroll
    for (int r = 0; r < SAMPLE_MAX_RANKS; ++r) {
      part[r] = 0;
      if (r < ranks)
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(part[r]) : "r"(sm_peer(&s.list_n, r)));
    }
#pragma unroll
    for (int r = 0; r < SAMPLE_MAX_RANKS; ++r) have += part[r];
#pragma unroll 1
    for (int i = tid; i < have; i += THREADS) {
      int from = 0, upto = 0, end = 0;
#pragma unroll
      for (int r = 0; r < SAMPLE_MAX_RANKS; ++r) {   // the rank that holds it, and its place there
        end += part[r];
        if (i >= end) { upto = end; from = r + 1; }   // (i < have: never behind the last)
      }
      float x;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(sm_peer(&s.list[i - upto], from)));
      s.all[i] = x;
      s.wall[i] = by_weight ? (unsigned long long)__double2ll_rn(weight(x) * unit) : 1ull;
    }
    __syncthreads();
    need *= unit;
    // `group` lanes to a token, each with some of those it is compared with; the
    // ranks share the tokens (and meet in an exchange, behind which the lists
    // may be filled anew)
    int lanes = 5;
    while (lanes > 0 && have << lanes > ranks * THREADS) --lanes;
    const int group = 1 << lanes;
    float best = -INFINITY;
    double above = 0.0;
#pragma unroll 1
    for (int i0 = 0; i0 < have; i0 += (ranks * THREADS) >> lanes) {
      const int i = i0 + ((rank * THREADS + tid) >> lanes);
      const float x = i < have ? s.all[i] : -INFINITY;
      unsigned long long gt = 0ull, eq = 0ull;
#pragma unroll 4
      for (int j = tid & (group - 1); j < have; j += group) {
        const unsigned long long w = s.wall[j];
        const float y = s.all[j];
        gt += y > x ? w : 0ull;
        eq += y == x ? w : 0ull;
      }
#pragma unroll 1
      for (int d = group / 2; d >= 1; d /= 2) {
        gt += __shfl_xor_sync(0xffffffffu, gt, d);
        eq += __shfl_xor_sync(0xffffffffu, eq, d);
      }
      if ((double)(gt + eq) >= need && x > best) { best = x; above = (double)gt; }
    }
    // the largest of the warp, of the CTA
#pragma unroll 1
    for (int d = 16; d >= 1; d /= 2) {
      const float y = __shfl_xor_sync(0xffffffffu, best, d);
      const double z = __shfl_xor_sync(0xffffffffu, above, d);
      if (y > best) { best = y; above = z; }
    }
    if (tid % 32 == 0) s.red[tid / 32] = {best, 0.0f, above, 0.0};
    __syncthreads();
    best = s.red[tid % (THREADS / 32)].x;
    above = s.red[tid % (THREADS / 32)].z;
#pragma unroll 1
    for (int d = THREADS / 64; d >= 1; d /= 2) {
      const float y = __shfl_xor_sync(0xffffffffu, best, d);
      const double z = __shfl_xor_sync(0xffffffffu, above, d);
      if (y > best) { best = y; above = z; }
    }
    const SampleShare* ex = sm_publish(s, ranks, rank, {best, 0.0f, above, 0.0});
    best = -INFINITY;
#pragma unroll 1
    for (int r = 0; r < ranks; ++r)
      if (ex[r].x > best) { best = ex[r].x; above = ex[r].z; }
    const double each = by_weight ? weight(best) * unit : 1.0;
    *ties = need - above <= each ? 1.0 : ceil((need - above) / each);    // (a division only where values repeat)
    return best;
  }

  // The border among the tokens of [lo, hi], `count` of them or fewer.
  // by_weight = false: the token of rank `goal`, from 1, from the largest down.
  // by_weight = true: the first token at which the running weight reaches
  // `goal`; n: count or weight above hi.  Returns its value; *ties: how many tokens
  // of that value are kept.
  __device__ __noinline__ float border(bool by_weight, float lo, float hi, int count, double goal, double n,
                                       double* ties) {
#pragma unroll 1
    for (int step = 0; step < 64 && lo < hi; ++step) {
      const Bins bins(lo, hi);
      open_bins();
      int b0 = 0, b1 = BINS - 1, left = count;
      if (count > SAMPLE_LIST) {
        sm_each(mine, run, [&](int, float x) {
          if (x >= lo && x <= hi) atomicAdd(&s.hist[bins.of(x)], 1u);
        });
        left = select_bins(by_weight, bins, lo, n, goal - (by_weight ? 0.0 : n), 0.0, &b0, &b1);
      }
      const bool listed = left <= SAMPLE_LIST;
      double above = 0.0;
      float top = -INFINITY, low = INFINITY;
      // (weights without a branch: those of several tokens overlap)
      sm_each<4>(mine, run, [&](int, float x) {
        const bool in = x >= lo && x <= hi;
        const int b = in ? bins.of(x) : BINS;
        const double v = by_weight ? weight(x) : 1.0;
        above += b < b0 ? v : 0.0;
        if (b < b0 || b > b1 || !in) return;
        top = fmaxf(top, x);
        low = fminf(low, x);
        if (listed) {
          const int at = atomicAdd(&s.list_n, 1);
          if (at < SAMPLE_LIST) s.list[at] = x;
        }
      });
      const SampleShare got = sm_combine<THREADS>(s, ranks, rank, {top, -low, above, 0.0});
      n += got.z;
      hi = got.x;
      lo = -got.y;
      count = left;
      if (!listed || !(lo < hi)) continue;
      const float best = pick(by_weight, fmax(goal - n, 0.0), ties);
      if (best > -INFINITY) return best;
      *ties = 1e18;                                  // (the goal is past them by a rounding)
      return lo;
    }
    // tokens of one value are left
    *ties = by_weight ? ceil((goal - n) / weight(hi)) : goal - n;
    return hi;
  }
};

// The draw among the tokens of one array, `count` of them at most in the
// cluster, all >= lo; `tail`: weight that top_p counts besides.  The index in it
// of the token, in one thread of the rank that holds it; -1 elsewhere.
template <typename T, int THREADS>
__device__ __noinline__ int sample_draw(Sampler<T, THREADS>& k, int per, float lo, int count, double tail,
                                        float u, int top_k, float top_p, float min_p) {
  SampleShared<T, THREADS>& sh = k.s;
  const int tid = k.tid, ranks = k.ranks, rank = k.rank, run = k.run;
  const T* mine = k.mine;
  // kept: x > tau, and the first `ties` of x = tau
  float tau = -INFINITY;
  double ties = 0.0;
  if (top_k > 0) {
    tau = k.border(false, lo, k.m, count, (double)top_k, 0.0, &ties);
    count = top_k;
    tail = 0.0;
  }
  if (top_p < 1.0f) {
    double w = 0.0, high = 0.0;                      // weight; of the tokens above `sure`
    float lowest = INFINITY;
    sm_each<4>(mine, run, [&](int, float x) {
      const double v = k.weight(x);
      w += x > tau ? v : 0.0;
      high += x > k.sure ? v : 0.0;
      lowest = fminf(lowest, x > tau ? x : INFINITY);
    });
    const SampleShare got = sm_combine<THREADS>(sh, ranks, rank, {-lowest, 0.0f, w, high});
    const double wt = tau == -INFINITY ? 0.0 : k.weight(tau);
    const double goal = fmax((double)top_p, 0.0) * (got.z + tail + ties * wt);
    if (tau > -INFINITY && goal > got.z) {           // inside the ties of top_k's border
      ties = fmin(ties, fmax(1.0, ceil((goal - got.z) / wt)));
    } else if (goal > 0.0) {
      // (not below m - 40 T, as above: an interval down to a mask's value, of which
      // the bins hold all weights in one, would not narrow)
      const float low = fmaxf(-got.x, (float)((double)k.m - 40.0 * 256.0 * 1.4426950408889634074 / k.c));
      const bool narrow = low < k.sure && k.sure < k.m;
      tau = k.border(true, low, narrow ? k.sure : k.m, count, goal, narrow ? got.w : 0.0, &ties);
      ties = fmax(ties, 1.0);
    } else {
      tau = k.m;                                     // the largest token at least
      ties = 1.0;
    }
  }

  // the kept tokens' weights and the ties of each run, and their running sums
  const double floor_w = fmin((double)min_p, 1.0);   // the largest token is always kept
  const bool has_floor = min_p > 0.0f;
  const double wt = tau == -INFINITY ? 0.0 : k.weight(tau);
  if (has_floor && wt < floor_w) ties = 0.0;
  SampleSums sum = {0.0, 0.0f, 0.0f}, all;       // kept weight, ties
  {
    const double least = has_floor ? floor_w : 0.0;
    int eq = 0;
    sm_each<4>(mine, run, [&](int, float x) {
      const double v = k.weight(x);
      eq += x == tau ? 1 : 0;
      sum.x += x > tau && v >= least ? v : 0.0;
    });
    sum.y = tau == -INFINITY ? 0.0f : (float)eq;
  }
  const SampleSums inc = sm_scan<THREADS>(sh, sum, &all);
  // (counts of ties are exact in a float: at most 2^24 tokens a rank)
  const SampleShare* ex = sm_publish(sh, ranks, rank, {all.y, 0.0f, all.x, 0.0});
  // the ranks in order: their weight, with the ties that are kept
  double total = 0.0, before = 0.0, eq0 = 0.0, seen = 0.0;
#pragma unroll 1
  for (int r = 0; r < ranks; ++r) {
    if (r == rank) { before = total; eq0 = seen; }
    total += ex[r].z + fmin(fmax(ties - seen, 0.0), (double)ex[r].x) * wt;
    seen += (double)ex[r].x;
  }
  const double goal = (u > 0.0f ? (double)fminf(u, 0.99999994f) : 0.0) * total;
  // the rank, and its first thread, whose running weight exceeds the goal
  double upto = 0.0;
  int who = 0;
  seen = 0.0;
#pragma unroll 1
  for (int r = 0; r < ranks; ++r) {
    const double own = ex[r].z + fmin(fmax(ties - seen, 0.0), (double)ex[r].x) * wt;
    upto += own;
    seen += (double)ex[r].x;
    if (own > 0.0) who = r;
    if (own > 0.0 && upto > goal) break;
  }
  if (who != rank) return -1;
  const double allowed = fmax(ties - eq0, 0.0);      // ties this rank may keep
  const double end = before + (inc.x + fmin(allowed, (double)inc.y) * wt);
  const double own = sum.x + (fmin(allowed, (double)inc.y) - fmin(allowed, (double)(inc.y - sum.y))) * wt;
  if (tid == 0) { sh.b0 = THREADS; sh.b1 = -1; }
  __syncthreads();
  if (own > 0.0) {
    if (end > goal) atomicMin(&sh.b0, tid);
    atomicMax(&sh.b1, tid);
  }
  __syncthreads();
  const int owner = sh.b0 < THREADS ? sh.b0 : sh.b1;
  if (owner < 0 || owner / 32 != tid / 32) return -1;
  // its warp looks through its run, 32 tokens at a time
  const int lane = tid % 32, src_lane = owner % 32;
  double sofar = __shfl_sync(0xffffffffu, end - own, src_lane);
  double seen_eq = __shfl_sync(0xffffffffu, eq0 + (double)(inc.y - sum.y), src_lane);
  const int len = __shfl_sync(0xffffffffu, run, src_lane);
  const T* runx = mine + (owner - tid) * per;
  int found = -1, last = 0;
#pragma unroll 1
  for (int i0 = 0; i0 < len && found < 0; i0 += 32) {
    const float x = i0 + lane < len ? to_f32(runx[i0 + lane]) : -INFINITY;
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
    const unsigned keep = __ballot_sync(0xffffffffu, v > 0.0);
    double acc = v;
#pragma unroll 1
    for (int d = 1; d < 32; d *= 2) {
      const double y = __shfl_up_sync(0xffffffffu, acc, d);
      if (lane >= d) acc += y;
    }
    const unsigned over = __ballot_sync(0xffffffffu, v > 0.0 && sofar + acc > goal);
    if (over) found = i0 + __ffs(over) - 1;
    if (keep) last = i0 + 31 - __clz(keep);
    sofar += __shfl_sync(0xffffffffu, acc, 31);
    seen_eq += (double)__popc(tied);
  }
  return lane == 0 ? owner * per + (found >= 0 ? found : last) : -1;
}

// The table of powers, before the kernel waits for the one ahead of it.
template <typename T, int THREADS>
__device__ __forceinline__ void sample_table(uint8_t* raw) {
  SampleShared<T, THREADS>& sh = *reinterpret_cast<SampleShared<T, THREADS>*>(raw);
  if (threadIdx.x < 256) sh.table[threadIdx.x] = exp2((double)threadIdx.x * (1.0 / 256.0));
}

// The token of a row (behind sample_table).
template <typename T, int THREADS>
__device__ __forceinline__ void sample_row(const SampleArgs& a, uint8_t* raw) {
  SampleShared<T, THREADS>& sh = *reinterpret_cast<SampleShared<T, THREADS>*>(raw);
  constexpr int VEC = 16 / sizeof(T);
  const int rank = blockIdx.x % a.ranks, row = blockIdx.x / a.ranks, tid = threadIdx.x;
  // every CTA of the cluster has started: waited for before the first store to
  // another's shared memory (a rank with few tokens or none gets there at once)
  if (a.ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int part = THREADS * a.run, base = rank * part;
  const int n = max(0, min(part, a.vocab - base));
  const T* src = static_cast<const T*>(a.logits) + row * a.row_stride + base;
  // 16-byte slots start after `head` tokens in memory; in shared memory they
  // are aligned too where that leaves the runs on whole words
  const int off = (int)((16u - (uint32_t)(reinterpret_cast<uintptr_t>(src) & 15u)) & 15u) / (int)sizeof(T);
  const int head = min(off, n);
  const bool wide = off % (4 / (int)sizeof(T)) == 0;
  T* xs = reinterpret_cast<T*>(raw + sizeof(SampleShared<T, THREADS>)) + (wide ? (VEC - off) % VEC : 0);
  if (tid == 0) sh.turn = 0;

  const float u = a.u[row];
  const float temperature = a.temperature ? a.temperature[row] : a.temperature_all;
  int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all;
  const float min_p = a.min_p ? a.min_p[row] : a.min_p_all;
  if (top_k >= a.vocab) top_k = 0;
  const bool filter = top_k > 0 || (top_p > 0.0f && top_p < 1.0f);

  // the tokens of this CTA; NaN as -inf, +inf as the largest finite value
  float top = -INFINITY, bottom = INFINITY;          // (of what is not -inf)
  int finite = 0;
  constexpr float MOST = sizeof(T) == 4 ? 3.402823466e38f
                         : std::is_same<T, bf16>::value ? 3.3895313892515355e38f : 65504.0f;
  auto clean = [&](T v) {
    const float x = fminf(fmaxf(to_f32(v), -INFINITY), MOST);    // (the maximum with NaN is the other)
    top = fmaxf(top, x);
    if (filter && x != -INFINITY) { bottom = fminf(bottom, x); ++finite; }
    return from_f32<T>(x);                           // (exact)
  };
  const int slots = (n - head) / VEC;
  constexpr int STEP = 4;                            // 16-byte loads in flight a thread
#pragma unroll 1
  for (int i0 = tid; i0 < slots; i0 += STEP * THREADS) {
    Slot<T, VEC> v[STEP];
#pragma unroll
    for (int j = 0; j < STEP; ++j) {
      const int i = i0 + j * THREADS;
      if (i < slots) v[j] = load_slot<kLoadStream, T, VEC>(src + head + i * VEC);
    }
#pragma unroll
    for (int j = 0; j < STEP; ++j) {
      const int i = i0 + j * THREADS;
      if (i >= slots) break;
#pragma unroll
      for (int q = 0; q < VEC; ++q) v[j].v[q] = clean(v[j].v[q]);
      T* dst = xs + head + i * VEC;
      if (wide) {
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(&v[j]);
      } else {
#pragma unroll
        for (int q = 0; q < VEC; ++q) dst[q] = v[j].v[q];
      }
    }
  }
  if (tid < head) xs[tid] = clean(src[tid]);
  const int behind = head + slots * VEC;
  if (behind + tid < n) xs[behind + tid] = clean(src[behind + tid]);   // (fewer than VEC)
  for (int i = n + tid; i < part; i += THREADS) xs[i] = from_f32<T>(-INFINITY);
  __syncthreads();

  Sampler<T, THREADS> k{sh, xs + tid * a.run, a.run, a.ranks, rank, tid, 0.0f, 0.0f, 0.0, INFINITY};
  const T* mine = k.mine;
  if (a.ranks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  const SampleShare range = sm_combine<THREADS>(sh, a.ranks, rank, {top, -bottom, (double)finite, 0.0});
  k.m = range.x;
  if (k.m == -INFINITY) {                            // nothing can be drawn
    if (rank == 0 && tid == 0) a.out[row] = -1;
    return;
  }
  if (!(temperature >= 1e-30f)) {                    // (1 / temperature stays a float)
    // (the first of the ranks' first indexes, as two halves of 16 bits)
    int at = 0x7fffffff;
    sm_each(mine, a.run, [&](int i, float x) {
      if (x == k.m) at = min(at, base + tid * a.run + i);
    });
    const float hi16 = (float)(at >> 16);
    const SampleShare first = sm_combine<THREADS>(sh, a.ranks, rank, {-hi16, 0.0f, 0.0, 0.0});
    const float lo16 = hi16 == -first.x ? (float)(at & 0xffff) : 65536.0f;
    const SampleShare second = sm_combine<THREADS>(sh, a.ranks, rank, {-lo16, 0.0f, 0.0, 0.0});
    if (rank == 0 && tid == 0) a.out[row] = ((int)-first.x << 16) + (int)-second.x;
    return;
  }
  k.c = 256.0 * 1.4426950408889634074 / (double)temperature;
  // e^-690 = 2^-995.  Rounded up: rounded down it can lie a whole step of m below
  // for 690 T of half a step, and the exponent of a weight at it leaves its field
  k.cut = fmaxf(__double2float_ru((double)k.m - 690.0 * (double)temperature), -3.402823466e38f);

  // `from`: what the filters keep is not below it
  float from = -INFINITY, lo = -range.y;
  const int count = (int)range.z;
  if (top_k >= count) top_k = 0;
  const bool by_weight = top_k <= 0;
  if (filter && (!by_weight || (top_p > 0.0f && top_p < 1.0f))) {
    // (weights below m - 40 T are under 5e-18 of the sum)
    if (by_weight) lo = fmaxf(lo, (float)((double)k.m - 40.0 * (double)temperature));
    from = lo;
    if (lo < k.m) {
      const SampleBins bins(lo, k.m);
      k.open_bins();
      sm_each(mine, a.run, [&](int, float x) {
        if (x >= lo) atomicAdd(&sh.hist[bins.of(x)], 1u);
      });
      int b0, b1;
      k.select_bins(by_weight, bins, lo, 0.0, by_weight ? -1.0 : (double)top_k, (double)top_p, &b0, &b1);
      // a little below the last bin's lower edge: its tokens are among the packed
      const float depth = ((float)b1 + 0.6f) * 2.0f / bins.inv;
      if (by_weight && b0 > 0) {
        const float height = ((float)b0 - 0.6f) * 2.0f / bins.inv;
        k.sure = (k.m - height) + 4e-7f * (fabsf(k.m) + height);         // (NaN past the range: no help)
      }
      if (b1 < SAMPLE_BINS - 1) from = fmaxf(lo, (k.m - depth) - 4e-7f * (fabsf(k.m) + depth));
    }
  }
  if (min_p > 0.0f && by_weight && !(top_p < 1.0f))  // (a little below its border)
    from = fmaxf(from, (float)((double)k.m + (log(fmin((double)min_p, 1.0)) - 1e-3) * (double)temperature) -
                           1e-6f * fabsf(k.m));

  int per = a.run, many = count;
  double tail = 0.0;
  bool packed = false, gather = false;
  if (from > -INFINITY) {
    // the tokens from there up; the weight of the rest
    int hits = 0;
    double rest = 0.0;
    if (by_weight && top_p < 1.0f)
      sm_each(mine, a.run, [&](int, float x) {
        hits += x >= from ? 1 : 0;
        const double w = k.weight(x);
        rest += x < from ? w : 0.0;
      });
    else
      sm_each(mine, a.run, [&](int, float x) { hits += x >= from ? 1 : 0; });
    SampleSums all;
    int place = (int)sm_scan<THREADS>(sh, {rest, (float)hits, 0.0f}, &all).y - hits;
    const SampleShare* ex = sm_publish(sh, a.ranks, rank, {0.0f, 0.0f, (double)all.y, all.x});
    int most = 0, first = 0;
    many = 0;
#pragma unroll 1
    for (int r = 0; r < a.ranks; ++r) {
      const int there = (int)ex[r].z;
      if (r == rank) first = many;
      if (tid == 0) sh.starts[r] = many;
      most = max(most, there);
      many += there;
      tail += ex[r].w;
    }
    // few: all to the first rank, which goes on alone; else each rank its own
    gather = many <= 4 * THREADS;
    packed = most <= sh.PACKED;
    if (packed) {
      const int target = gather ? 0 : rank, here = gather ? many : (int)all.y;
      if (gather) place += first;
      const uint32_t values = sm_peer(sh.packed, target), places = sm_peer(sh.packed_at, target);
      sm_few(mine, a.run, [&](float x) { return x >= from; }, [&](int i, float x) {
        sm_put(values, place, from_f32<T>(x));
        sm_put(places, place, (unsigned short)(tid * a.run + i));
        ++place;
      });
      constexpr int WORD = 4 / (int)sizeof(T);       // (runs of whole words: -inf behind the last)
      if (WORD == 2 && tid == 0 && rank == target && here % 2 != 0) sh.packed[here] = from_f32<T>(-INFINITY);
      if (gather) {
        sm_sync(a.ranks);
        if (rank != 0) return;
        k.ranks = 1;
      } else {
        __syncthreads();
      }
      per = ((here + THREADS - 1) / THREADS + WORD - 1) / WORD * WORD;
      k.mine = sh.packed + tid * per;
      k.run = max(0, min(per, (here + WORD - 1) / WORD * WORD - tid * per));
      lo = from;
    }
  }
  if (!packed) {                                     // the whole row, its tail included
    many = count;
    tail = 0.0;
  }
  const int at = sample_draw<T, THREADS>(k, per, lo, many, tail, u, top_k, top_p, min_p);
  if (at < 0) return;                                // (one thread has it: the largest token weighs 1 and is kept)
  int token = base + at;
  if (packed) {
    int r = rank;
    if (gather)
      for (r = a.ranks - 1; sh.starts[r] > at; --r) {}         // (starts[0] = 0)
    token = r * part + (int)sh.packed_at[at];
  }
  a.out[row] = token;
}

}  // namespace molten
