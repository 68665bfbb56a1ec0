// Attention of a few query rows over a sliding window and the first keys:
//
//   query i of request b stands at p = len_b - nq + i and sees key j iff
//   j <= p and (j > p - window or j < sinks);  o = softmax(q k^T scale) v
//   over the keys it sees, 0 if it sees none.
//
// For single tokens and a few speculated ones: the rows of a key head (nq
// queries times the heads that share it) number 8 NB at most, and each key
// and value is used only that often.  Bound by HBM: the keys and values that
// any query sees, read once.  The products run on mma.sync m16n8k16 (tcgen05
// would want 128 rows, and P written back to TMEM, for a result that is
// mostly padding) in the orientation whose narrow side is the rows: S^T = K
// Q^T and O^T = V^T P^T, with keys and head dims as the 16-row operands.  (With
// the rows as the 16-row operand half of every MMA was padding, and MMAs, not
// loads, bounded a warp: 1.0 us a tile.)  The S^T accumulators become the P^T
// operand by an 8 x 8 transposition (movmatrix).
//
// A warp owns tiles of 16 keys: it copies them with 16-byte cp.async into a
// ring of its own (no barrier between warps; STAGES - 1 tiles in flight),
// keeps the running maximum and sum of its rows in fp32, and at the end the
// warps of a CTA, the CTAs of a cluster (through distributed shared memory)
// and, where even that leaves SMs idle, the parts of a long cache (a second
// small kernel) are joined by the usual rescaling.
//
// P is the sum of two 16-bit values (P and what its rounding leaves), two
// MMAs: P V is exact to 2^-16, so the output rounding is the only one that
// shows, and the second MMA hides behind the loads.  fp16 weights (and with them
// O and the sum) are taken times 2^15: their largest is 2^15, and the two parts
// keep their bits down to 2^-28 of it (without: down to 2^-13, nothing below 2^-25).
//
// Keys that no query sees are not read: their slots are zero-filled, so
// whatever a cache holds behind its last token or outside the window never
// meets an MMA.  A key that only some queries see takes part with P = 0; if
// its value holds an infinity or NaN (0 times that is NaN) the tile's P V is
// done row by row instead.  A warp whose sums end with an infinity or NaN takes
// its tiles once more, all of them row by row: the two parts of P times an
// infinity can be infinities of both signs.
//
// Measured: 64 requests over caches of up to 8192, 32 heads over 8, head dim
// 128, window 4096: 156 us, 6.9 TB/s of the keys and values that are seen (167 and
// 6.4 at the clock that seconds of such calls leave); 1 request over 4096, window
// 1024: 6.8 us, of it some 4 the latency of a launch,
// the first loads and the exchange of the cluster.
#pragma once

#include "molten/common.cuh"

namespace molten {

struct WindowArgs {
  const void* q;                   // [batch, nq, kv_heads * per, dim]
  const void* k;                   // [batch, cache, kv_heads, dim]
  const void* v;
  const int* lengths;              // [batch] valid keys, or null: cache
  void* out;                       // [batch, nq, heads, dim] contiguous
  float* part;                     // [item][part][rows][dim + 2] partial results (parts > 1)
  long long q_b, q_s, q_h, k_b, k_s, k_h, v_b, v_s, v_h;   // strides in elements
  int batch, nq, cache, kv_heads, per, dim;
  int window, sinks;               // window < 0: every earlier key
  float scale_log2;                // scale * log2(e)
  int ranks, parts;                // CTAs of the cluster; clusters per item
  int reserved;
};

__device__ __forceinline__ uint32_t wd_smem(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void wd_copy16(uint32_t dst, const void* src, bool in) {
  const int n = in ? 16 : 0;                         // 0: zero-filled, nothing read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(n) : "memory");
}
template <bool TRANS>
__device__ __forceinline__ void wd_ldmatrix(uint32_t addr, uint32_t (&r)[4]) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void wd_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, f16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t wd_pack(float x, float y) {
  Slot<T, 2> s;
  const float f[2] = {x, y};
  pack_slot<T, 2>(s, f);
  return *reinterpret_cast<const uint32_t*>(&s);
}
template <typename T> __device__ __forceinline__ float2 wd_unpack(uint32_t u) {
  const Slot<T, 2> s = *reinterpret_cast<const Slot<T, 2>*>(&u);
  return make_float2(to_f32(s.v[0]), to_f32(s.v[1]));
}

// The keys that some query of the request sees: [0, sink) and [start, len),
// as tiles of TILE keys; sink tiles first.
struct WindowSpan {
  int len, first, last;            // keys; positions of the first and last query
  int start;                       // first key of the first query's window
  int sink_tiles, start_tile, tiles;
  template <int TILE>
  __device__ __forceinline__ static WindowSpan of(const WindowArgs& a, int b) {
    WindowSpan s;
    int n = a.lengths ? a.lengths[b] : a.cache;
    n = n < 0 ? 0 : (n > a.cache ? a.cache : n);
    s.len = n;
    s.last = n - 1;
    s.first = n - a.nq;
    const int p = s.first > 0 ? s.first : 0;
    s.start = a.window < 0 || p < a.window ? 0 : p - a.window + 1;
    s.start_tile = s.start / TILE;
    const int end = (n + TILE - 1) / TILE;
    const int sink = (min(a.sinks, n) + TILE - 1) / TILE;
    s.sink_tiles = min(sink, s.start_tile);
    s.tiles = s.sink_tiles + end - s.start_tile;
    return s;
  }
  template <int TILE> __device__ __forceinline__ int key0(int tile) const {
    return (tile < sink_tiles ? tile : tile - sink_tiles + start_tile) * TILE;
  }
  __device__ __forceinline__ bool any(const WindowArgs& a, int j) const {
    return j < len && (j >= start || j < a.sinks);
  }
  __device__ __forceinline__ bool sees(const WindowArgs& a, int p, int j) const {
    return j <= p && (a.window < 0 || j > p - a.window || j < a.sinks);
  }
};

// z: (x, y, maximum, sum) of one share of a row's keys, joined with another's.
__device__ __forceinline__ void wd_join(float4& z, const float4& w) {
  if (w.z == -INFINITY && w.w == 0.0f) return;       // saw no key
  const float mn = fmaxf(z.z, w.z);
  const float f0 = fast_exp2(z.z - mn), f1 = fast_exp2(w.z - mn);
  z.w = z.w * f0 + w.w * f1;
  z.x = z.x * f0 + w.x * f1;
  z.y = z.y * f0 + w.y * f1;
  z.z = mn;
}

// Columns d and d + 1 of row r: the output, or the part's share of it.
template <typename OT>
__device__ __forceinline__ void window_store(const WindowArgs& a, int b, int h, int item, int part,
                                             int rows, int r, int d, const float4& z) {
  if (a.parts == 1) {
    const float inv = z.w == 0.0f ? 0.0f : 1.0f / z.w;
    const int q = r / a.per, hd = h * a.per + r % a.per;
    OT* dst = static_cast<OT*>(a.out) +
              (((long long)b * a.nq + q) * (a.kv_heads * a.per) + hd) * a.dim + d;
    Slot<OT, 2> so;
    const float f[2] = {z.x * inv, z.y * inv};
    pack_slot<OT, 2>(so, f);
    *reinterpret_cast<Slot<OT, 2>*>(dst) = so;
  } else {
    float* dst = a.part + (((long long)item * a.parts + part) * rows + r) * (a.dim + 2);
    *reinterpret_cast<float2*>(dst + d) = make_float2(z.x, z.y);
    if (d == 0) *reinterpret_cast<float2*>(dst + a.dim) = make_float2(z.z, z.w);
  }
}

__device__ __forceinline__ uint32_t wd_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// DP: dim padded to 64 or 128.  NB: blocks of 8 rows.
template <int DP, int NB, int WARPS, int STAGES>
struct WindowDecodeLayout {
  static constexpr int TILE = 16, ROWS = 8 * NB;
  static constexpr int KV_BYTES = TILE * DP * 2;     // one tile of K or V
  static constexpr int RING = WARPS * STAGES * 2 * KV_BYTES;
  static constexpr int OUT = WARPS * ROWS * (DP + 4) * 4;       // merge area (over the ring)
  static constexpr int STAT = WARPS * ROWS * 8;
  static constexpr int PROB = WARPS * ROWS * TILE * 4;
  static constexpr int SMEM = (RING > OUT ? RING : OUT) + STAT + PROB;
};

template <typename T, typename OT, int DP, int NB, int WARPS, int STAGES>
__device__ __forceinline__ void window_decode(const WindowArgs& a, uint8_t* raw) {
  typedef WindowDecodeLayout<DP, NB, WARPS, STAGES> L;
  constexpr int TILE = L::TILE, ROWS = L::ROWS, NK = DP / 16, PITCH = DP * 2;
  constexpr int CHUNKS = DP / 8;                     // 16-byte chunks of a row
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane / 4, t = lane % 4;
  const int rank = blockIdx.x % a.ranks, rest0 = blockIdx.x / a.ranks;
  const int part = rest0 % a.parts, item = rest0 / a.parts;
  const int b = item / a.kv_heads, h = item - b * a.kv_heads;
  const int rows = a.nq * a.per;
  if (a.ranks > 1)                                   // every CTA of the cluster has started: waited
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");     // for before the merge

  // Q^T as B operands (row n of a block is lane group g); row r is query
  // r / per, head r % per.  A lane keeps statistics of rows 2 t, 2 t + 1.
  uint32_t qb[NB][NK][2];
  int pos[NB][2];                                    // where those two rows stand
#pragma unroll
  for (int n = 0; n < NB; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = n * 8 + 2 * t + e;
      pos[n][e] = r < rows ? r / a.per : -0x40000000;
    }
    const int r = n * 8 + g, i = min(r / a.per, a.nq - 1);
    const T* src = static_cast<const T*>(a.q) + b * a.q_b + (long long)i * a.q_s
                   + (long long)(h * a.per + r % a.per) * a.q_h;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int d = k * 16 + c * 8 + 2 * t;
        qb[n][k][c] = r < rows && d < a.dim ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
      }
    }
  }
  const WindowSpan span = WindowSpan::of<TILE>(a, b);
#pragma unroll
  for (int n = 0; n < NB; ++n) { pos[n][0] += span.first; pos[n][1] += span.first; }
  // tiles of this CTA: an equal share of the item's, in order
  const int shares = a.ranks * a.parts, share = part * a.ranks + rank;
  const int t0 = (int)((long long)span.tiles * share / shares);
  const int t1 = (int)((long long)span.tiles * (share + 1) / shares);

  const T* kb = static_cast<const T*>(a.k) + b * a.k_b + h * a.k_h;
  const T* vb = static_cast<const T*>(a.v) + b * a.v_b + h * a.v_h;
  uint8_t* ring = raw + warp * (STAGES * 2 * L::KV_BYTES);
  const uint32_t ring_s = wd_smem(ring);
  float* stat = reinterpret_cast<float*>(raw + (L::RING > L::OUT ? L::RING : L::OUT));
  float* prob = stat + WARPS * ROWS * 2 + warp * ROWS * TILE;

  // a lane copies chunk cc of every RSTEP-th row of a tile
  constexpr int RSTEP = 32 / CHUNKS;
  const int cc = lane % CHUNKS, cr = lane / CHUNKS;
  const bool col = cc * 8 < a.dim;                   // chunks past the head dim are zero-filled
  const T* kl = kb + (col ? cc * 8 : 0);
  const T* vl = vb + (col ? cc * 8 : 0);
  auto copy_tile = [&](int tile, int stage) {
    if (tile < t1) {
      const int key0 = span.key0<TILE>(tile) + cr;
      const uint32_t dst = ring_s + stage * (2 * L::KV_BYTES);
      const T* ks = kl + (long long)key0 * a.k_s;
      const T* vs = vl + (long long)key0 * a.v_s;
      const int last = key0 - cr + TILE - 1;
      const bool full = last < span.len && (key0 - cr >= span.start || last < a.sinks);
#pragma unroll
      for (int i = 0; i < TILE / RSTEP; ++i) {
        const int r = cr + i * RSTEP;
        const bool in = col && (full || span.any(a, key0 + i * RSTEP));
        const uint32_t off = r * PITCH + ((cc ^ (r & 7)) << 4);
        // (nothing is read where nothing is wanted; the address stays valid)
        wd_copy16(dst + off, in ? ks : kb, in);
        wd_copy16(dst + L::KV_BYTES + off, in ? vs : vb, in);
        ks += RSTEP * a.k_s;
        vs += RSTEP * a.v_s;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  float o[NB][NK][4], mx[NB][2], sum[NB][2];         // O^T: dims 16 i + g, + 8; rows 2 t, 2 t + 1
  // a second turn, with every tile done row by row, where the first left a NaN
#pragma unroll 1
  for (int turn = 0; turn < 2; ++turn) {
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) copy_tile(t0 + warp + s * WARPS, s);
#pragma unroll
  for (int n = 0; n < NB; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) { mx[n][e] = -INFINITY; sum[n][e] = 0.0f; }
#pragma unroll
    for (int i = 0; i < NK; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][i][e] = 0.0f;
  }

  int stage = 0;
#pragma unroll 1
  for (int tile = t0 + warp; tile < t1; tile += WARPS) {
    {
      int next = stage + STAGES - 1;
      if (next >= STAGES) next -= STAGES;
      copy_tile(tile + (STAGES - 1) * WARPS, next);
    }
    asm volatile("cp.async.wait_group %0;" :: "n"(STAGES - 1) : "memory");
    __syncwarp();
    const int key0 = span.key0<TILE>(tile);
    const uint32_t ks = ring_s + stage * (2 * L::KV_BYTES), vs = ks + L::KV_BYTES;
    const uint8_t* vt = ring + stage * (2 * L::KV_BYTES) + L::KV_BYTES;

    // S^T: keys g, g + 8; rows 2 t, 2 t + 1; even and odd steps in chains of their own
    float s[NB][4], s2[NB][4];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) { s[n][e] = 0.0f; s2[n][e] = 0.0f; }
    const int kr = (lane & 7) + (((lane >> 3) & 1) << 3), kc = lane >> 4;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      uint32_t kf[4];
      wd_ldmatrix<false>(ks + kr * PITCH + (((2 * k + kc) ^ (kr & 7)) << 4), kf);
#pragma unroll
      for (int n = 0; n < NB; ++n) wd_mma<T>(k % 2 ? s2[n] : s[n], kf, qb[n][k][0], qb[n][k][1]);
    }

    // keys that every query sees need no mask
    const bool whole = key0 + TILE - 1 <= span.first &&
                       (a.window < 0 || key0 > span.last - a.window || key0 + TILE <= a.sinks);
    uint32_t ph[NB][2], pl[NB][2];
    float fix[NB][2];
    bool moved = false;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {                  // rows 2 t, 2 t + 1
        float x0 = (s[n][e] + s2[n][e]) * a.scale_log2;
        float x1 = (s[n][e + 2] + s2[n][e + 2]) * a.scale_log2;
        if (!whole) {
          if (!span.sees(a, pos[n][e], key0 + g)) x0 = -INFINITY;
          if (!span.sees(a, pos[n][e], key0 + g + 8)) x1 = -INFINITY;
        }
        float top = fmaxf(x0, x1);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const float mn = fmaxf(mx[n][e], top);
        const float base = mn == -INFINITY ? 0.0f : mn;
        fix[n][e] = fast_exp2(mx[n][e] - base);
        moved |= mn != mx[n][e];
        mx[n][e] = mn;
        x0 -= base;
        x1 -= base;
        if constexpr (std::is_same<T, f16>::value) { x0 += 15.0f; x1 += 15.0f; }
        x0 = fast_exp2(x0);
        x1 = fast_exp2(x1);
        sum[n][e] = sum[n][e] * fix[n][e] + (x0 + x1);
        s[n][e] = x0;
        s[n][e + 2] = x1;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {                  // keys 0..7, 8..15
        const uint32_t hi = wd_pack<T>(s[n][2 * c], s[n][2 * c + 1]);
        const float2 hf = wd_unpack<T>(hi);
        ph[n][c] = wd_transpose(hi);
        pl[n][c] = wd_transpose(wd_pack<T>(s[n][2 * c] - hf.x, s[n][2 * c + 1] - hf.y));
      }
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          o[n][i][0] *= fix[n][0]; o[n][i][1] *= fix[n][1];
          o[n][i][2] *= fix[n][0]; o[n][i][3] *= fix[n][1];
        }
    }

    bool odd = turn > 0;                             // an infinity or NaN that P = 0 would meet
    if (a.nq > 1 && !whole && !odd) {
#pragma unroll 1
      for (int i = lane; i < L::KV_BYTES / 4; i += 32) {
        const float2 f = wd_unpack<T>(*reinterpret_cast<const uint32_t*>(vt + 4 * i));
        odd |= !isfinite(f.x) || !isfinite(f.y);
      }
      odd = __any_sync(0xffffffffu, odd);
    }
    if (!odd) {
      const int vm = lane >> 3, vr = (lane & 7) + ((vm >> 1) << 3), vc = vm & 1;
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        uint32_t vf[4];
        wd_ldmatrix<true>(vs + vr * PITCH + (((2 * i + vc) ^ (vr & 7)) << 4), vf);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          wd_mma<T>(o[n][i], vf, ph[n][0], ph[n][1]);
          wd_mma<T>(o[n][i], vf, pl[n][0], pl[n][1]);
        }
      }
    } else {
      // row by row, over the keys each row sees
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          prob[(n * 8 + 2 * t + (e & 1)) * TILE + g + (e >> 1) * 8] = s[n][e];
      __syncwarp();
#pragma unroll 1
      for (int kk = 0; kk < TILE; ++kk) {
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          const T* row = reinterpret_cast<const T*>(vt + kk * PITCH);
          const float v0 = to_f32(row[(((2 * i) ^ (kk & 7)) << 3) + g]);
          const float v1 = to_f32(row[(((2 * i + 1) ^ (kk & 7)) << 3) + g]);
#pragma unroll
          for (int n = 0; n < NB; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (!span.sees(a, pos[n][e], key0 + kk)) continue;
              const float p = prob[(n * 8 + 2 * t + e) * TILE + kk];
              o[n][i][e] += p * v0;
              o[n][i][e + 2] += p * v1;
            }
          }
        }
      }
    }
    __syncwarp();                                    // the stage is free for the next copy
    if (++stage == STAGES) stage = 0;
  }
  // 0 x sums up to NaN from an infinity or NaN on: P's two parts times an
  // infinity may be infinities of both signs
  float odds[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int i = 0; i < NK; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) odds[e] = fmaf(o[n][i][e], 0.0f, odds[e]);
  odds[0] = (odds[0] + odds[1]) + (odds[2] + odds[3]);
  if (!__any_sync(0xffffffffu, odds[0] != odds[0])) break;
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();                                   // every ring is idle: the merge area

  // each warp's rows: maximum and sum, O
  float* area = reinterpret_cast<float*>(raw);
  constexpr int OP = DP + 4;                         // pitch (rows on different banks)
#pragma unroll
  for (int n = 0; n < NB; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float total = sum[n][e];
      total += __shfl_xor_sync(0xffffffffu, total, 4);
      total += __shfl_xor_sync(0xffffffffu, total, 8);
      total += __shfl_xor_sync(0xffffffffu, total, 16);
      const int r = n * 8 + 2 * t + e;
      if (r >= rows) continue;
      if (g == 0) {
        stat[(warp * ROWS + r) * 2] = mx[n][e];
        stat[(warp * ROWS + r) * 2 + 1] = total;
      }
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        area[(warp * ROWS + r) * OP + i * 16 + g] = o[n][i][e];
        area[(warp * ROWS + r) * OP + i * 16 + g + 8] = o[n][i][e + 2];
      }
    }
  }
  __syncthreads();

  // a (row, 2 columns) pair a thread: join the CTA's warps in order; with a
  // cluster, push the result to the rank that owns the pair
  const int pairs = a.dim / 2, total = rows * pairs;
  const int own = (total + a.ranks - 1) / a.ranks;   // pairs of one rank
  float4* inbox = reinterpret_cast<float4*>(raw + L::SMEM);      // [rank][own]
  if (a.ranks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
#pragma unroll 1
  for (int i = threadIdx.x; i < total; i += WARPS * 32) {
    const int r = i / pairs, d = (i - r * pairs) * 2;
    float2 ms[WARPS], v[WARPS];
    float4 z = make_float4(0.0f, 0.0f, -INFINITY, 0.0f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      ms[w] = *reinterpret_cast<const float2*>(&stat[(w * ROWS + r) * 2]);
      v[w] = *reinterpret_cast<const float2*>(&area[(w * ROWS + r) * OP + d]);
    }
#pragma unroll
    for (int w = 0; w < WARPS; ++w) wd_join(z, make_float4(v[w].x, v[w].y, ms[w].x, ms[w].y));
    if (a.ranks == 1) {
      window_store<OT>(a, b, h, item, part, rows, r, d, z);
    } else {
      const int owner = i / own;
      uint32_t at = wd_smem(inbox + rank * own + (i - owner * own));
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(at), "r"(owner));
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};"
                   :: "r"(at), "f"(z.x), "f"(z.y), "f"(z.z), "f"(z.w) : "memory");
    }
  }
  if (a.ranks > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
#pragma unroll 1
    for (int i = threadIdx.x; i < own && rank * own + i < total; i += WARPS * 32) {
      float4 x[8];                                   // at most 8 ranks
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < a.ranks) x[c] = inbox[c * own + i];
      float4 z = make_float4(0.0f, 0.0f, -INFINITY, 0.0f);
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < a.ranks) wd_join(z, x[c]);
      const int at = rank * own + i, r = at / pairs, d = (at - r * pairs) * 2;
      window_store<OT>(a, b, h, item, part, rows, r, d, z);
    }
  }
}

// Join the parts of every row: a warp per (item, row).
template <typename OT>
__device__ __forceinline__ void window_join(const WindowArgs& a) {
  const int rows = a.nq * a.per;
  const long long total = (long long)a.batch * a.kv_heads * rows;
  const long long id = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  if (id >= total) return;
  const int lane = threadIdx.x % 32;
  const long long item = id / rows;
  const int r = (int)(id - item * rows);
  const int b = (int)(item / a.kv_heads), h = (int)(item - (long long)b * a.kv_heads);
  const long long pitch = a.dim + 2, step = (long long)rows * pitch;
  const float* src = a.part + item * a.parts * step + r * pitch;
  float M = -INFINITY;
  for (int p = 0; p < a.parts; ++p) {
    const float2 ms = *reinterpret_cast<const float2*>(src + p * step + a.dim);
    if (ms.y != 0.0f) M = fmaxf(M, ms.x);
  }
  float S = 0.0f;
  for (int p = 0; p < a.parts; ++p) {
    const float2 ms = *reinterpret_cast<const float2*>(src + p * step + a.dim);
    if (ms.y != 0.0f) S += ms.y * fast_exp2(ms.x - M);
  }
  const float inv = S == 0.0f ? 0.0f : 1.0f / S;
  const int q = r / a.per, hd = h * a.per + r % a.per;
  OT* dst = static_cast<OT*>(a.out) + (((long long)b * a.nq + q) * (a.kv_heads * a.per) + hd) * a.dim;
  for (int d = 2 * lane; d < a.dim; d += 64) {
    float x = 0.0f, y = 0.0f;
    for (int p = 0; p < a.parts; ++p) {
      const float2 ms = *reinterpret_cast<const float2*>(src + p * step + a.dim);
      if (ms.y == 0.0f) continue;
      const float f = fast_exp2(ms.x - M);
      const float2 v = *reinterpret_cast<const float2*>(src + p * step + d);
      x += v.x * f;
      y += v.y * f;
    }
    Slot<OT, 2> so;
    const float f[2] = {x * inv, y * inv};
    pack_slot<OT, 2>(so, f);
    *reinterpret_cast<Slot<OT, 2>*>(dst + d) = so;
  }
}

}  // namespace molten
