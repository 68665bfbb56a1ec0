// Attention of a few query rows over a sliding window and the first keys:
//
//   query i of request b stands at p = len_b - nq + i and sees key j iff
//   j <= p and (j > p - window or j < sinks);  o = softmax(q k^T scale) v
//   over the keys it sees, 0 if it sees none.
//
// For single tokens and a few speculated ones: the rows of a key head (nq
// queries times the heads that share it, at most 16 MT) fit one or two MMA
// row tiles, and each key and value is used only that often.  Bound by HBM:
// the keys and values that any query sees, read once.  So loads decide and
// the products run on mma.sync m16n8k16, whose S accumulators are the A
// operand of P V as they stand (tcgen05 would want 128 rows and P written
// back to TMEM for a result that is mostly padding).
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
// shows, and the second MMA hides behind the loads.
//
// Keys that no query sees are not read: their slots are zero-filled, so
// whatever a cache holds behind its last token or outside the window never
// meets an MMA.  A key that only some queries see takes part with P = 0; if
// its value holds an infinity or NaN (0 times that is NaN) the tile's P V is
// done row by row instead.
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

// DP: dim padded to 64 or 128.
template <int DP, int MT, int WARPS, int STAGES>
struct WindowDecodeLayout {
  static constexpr int TILE = 16, ROWS = 16 * MT;
  static constexpr int KV_BYTES = TILE * DP * 2;     // one tile of K or V
  static constexpr int RING = WARPS * STAGES * 2 * KV_BYTES;
  static constexpr int OUT = WARPS * ROWS * (DP + 4) * 4;       // merge area (over the ring)
  static constexpr int STAT = WARPS * ROWS * 8;
  static constexpr int PROB = WARPS * ROWS * TILE * 4;
  static constexpr int SMEM = (RING > OUT ? RING : OUT) + STAT + PROB;
};

template <typename T, typename OT, int DP, int MT, int WARPS, int STAGES>
__device__ __forceinline__ void window_decode(const WindowArgs& a, uint8_t* raw) {
  typedef WindowDecodeLayout<DP, MT, WARPS, STAGES> L;
  constexpr int TILE = L::TILE, ROWS = L::ROWS, NK = DP / 16, ND = DP / 8, PITCH = DP * 2;
  constexpr int CHUNKS = DP / 8;                     // 16-byte chunks of a row
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane / 4, t = lane % 4;
  const int rank = blockIdx.x % a.ranks, rest0 = blockIdx.x / a.ranks;
  const int part = rest0 % a.parts, item = rest0 / a.parts;
  const int b = item / a.kv_heads, h = item - b * a.kv_heads;
  const int rows = a.nq * a.per;
  const WindowSpan span = WindowSpan::of<TILE>(a, b);
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

  auto copy_tile = [&](int tile, int stage) {
    if (tile < t1) {
      const int key0 = span.key0<TILE>(tile);
      const uint32_t dst = ring_s + stage * (2 * L::KV_BYTES);
#pragma unroll
      for (int i = 0; i < TILE * CHUNKS / 32; ++i) {
        const int c = (i * 32 + lane) % CHUNKS, r = (i * 32 + lane) / CHUNKS;
        const int j = key0 + r;
        const bool in = span.any(a, j) && c * 8 < a.dim;
        const long long jj = in ? j : 0;
        const int cc = in ? c * 8 : 0;
        const uint32_t off = r * PITCH + ((c ^ (r & 7)) << 4);
        wd_copy16(dst + off, kb + jj * a.k_s + cc, in);
        wd_copy16(dst + L::KV_BYTES + off, vb + jj * a.v_s + cc, in);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) copy_tile(t0 + warp + s * WARPS, s);

  // the rows of q as A operands; row r is query r / per, head r % per
  uint32_t qa[MT][NK][4];
  int pos[MT][2];                                    // where rows g and g + 8 stand
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = m * 16 + e * 8 + g;
      const int i = r / a.per;
      pos[m][e] = r < rows ? span.first + i : -1;
      const T* src = static_cast<const T*>(a.q) + b * a.q_b + (long long)min(i, a.nq - 1) * a.q_s
                     + (long long)(h * a.per + r % a.per) * a.q_h;
#pragma unroll
      for (int k = 0; k < NK; ++k) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int d = k * 16 + c * 8 + 2 * t;
          qa[m][k][c * 2 + e] = r < rows && d < a.dim ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
        }
      }
    }
  }

  float o[MT][ND][4], mx[MT][2], sum[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int e = 0; e < 2; ++e) { mx[m][e] = -INFINITY; sum[m][e] = 0.0f; }
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[m][n][e] = 0.0f;
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
    const int kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;

    float s[MT][2][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[m][n][e] = 0.0f;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      uint32_t kf[4];
      wd_ldmatrix<false>(ks + kr * PITCH + (((2 * k + kc) ^ (kr & 7)) << 4), kf);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        wd_mma<T>(s[m][0], qa[m][k], kf[0], kf[1]);
        wd_mma<T>(s[m][1], qa[m][k], kf[2], kf[3]);
      }
    }

    // keys that every query sees need no mask
    const bool whole = key0 + TILE - 1 <= span.first &&
                       (a.window < 0 || key0 > span.last - a.window || key0 + TILE <= a.sinks);
    uint32_t ph[MT][4], pl[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {                  // rows g, g + 8
        float x[4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int j = key0 + n * 8 + 2 * t + c;
            const float v = s[m][n][e * 2 + c] * a.scale_log2;
            x[n * 2 + c] = whole || span.sees(a, pos[m][e], j) ? v : -INFINITY;
          }
        float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float mn = fmaxf(mx[m][e], top);
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float fix = fast_exp2(mx[m][e] - base);
        if (__any_sync(0xffffffffu, mn != mx[m][e])) {
          sum[m][e] *= fix;
#pragma unroll
          for (int n = 0; n < ND; ++n) { o[m][n][e * 2] *= fix; o[m][n][e * 2 + 1] *= fix; }
        }
        mx[m][e] = mn;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          x[q] = fast_exp2(x[q] - base);
          sum[m][e] += x[q];
          s[m][q / 2][e * 2 + q % 2] = x[q];
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint32_t hi = wd_pack<T>(x[2 * n], x[2 * n + 1]);
          const float2 hf = wd_unpack<T>(hi);
          ph[m][n * 2 + e] = hi;
          pl[m][n * 2 + e] = wd_pack<T>(x[2 * n] - hf.x, x[2 * n + 1] - hf.y);
        }
      }
    }

    bool odd = false;                                // an infinity or NaN that P = 0 would meet
    if (a.nq > 1 && !whole) {
#pragma unroll 1
      for (int i = lane; i < L::KV_BYTES / 4; i += 32) {
        const uint32_t u = *reinterpret_cast<const uint32_t*>(ring + stage * (2 * L::KV_BYTES) +
                                                              L::KV_BYTES + 4 * i);
        const float2 f = wd_unpack<T>(u);
        odd |= !isfinite(f.x) || !isfinite(f.y);
      }
      odd = __any_sync(0xffffffffu, odd);
    }
    if (!odd) {
      const int vr = (lane & 7) + (((lane >> 3) & 1) << 3), vc = lane >> 4;
#pragma unroll
      for (int n = 0; n < ND / 2; ++n) {
        uint32_t vf[4];
        wd_ldmatrix<true>(vs + vr * PITCH + (((2 * n + vc) ^ (vr & 7)) << 4), vf);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          wd_mma<T>(o[m][2 * n], ph[m], vf[0], vf[1]);
          wd_mma<T>(o[m][2 * n + 1], ph[m], vf[2], vf[3]);
          wd_mma<T>(o[m][2 * n], pl[m], vf[0], vf[1]);
          wd_mma<T>(o[m][2 * n + 1], pl[m], vf[2], vf[3]);
        }
      }
    } else {
      // row by row, over the keys each row sees
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            prob[(m * 16 + g + (e >> 1) * 8) * TILE + n * 8 + 2 * t + (e & 1)] = s[m][n][e];
      __syncwarp();
#pragma unroll 1
      for (int kk = 0; kk < TILE; ++kk) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float p = prob[(m * 16 + g + e * 8) * TILE + kk];
            if (!span.sees(a, pos[m][e], key0 + kk)) continue;
#pragma unroll
            for (int n = 0; n < ND; ++n) {
              const uint32_t u = *reinterpret_cast<const uint32_t*>(
                  ring + stage * (2 * L::KV_BYTES) + L::KV_BYTES + kk * PITCH + ((n ^ (kk & 7)) << 4) + 4 * t);
              const float2 f = wd_unpack<T>(u);
              o[m][n][e * 2] += p * f.x;
              o[m][n][e * 2 + 1] += p * f.y;
            }
          }
        }
      }
    }
    __syncwarp();                                    // the stage is free for the next copy
    if (++stage == STAGES) stage = 0;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();                                   // every ring is idle: the merge area

  // each warp's rows: maximum and sum, O
  float* area = reinterpret_cast<float*>(raw);
  constexpr int OP = DP + 4;                         // pitch (rows on different banks)
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float total = sum[m][e];
      total += __shfl_xor_sync(0xffffffffu, total, 1);
      total += __shfl_xor_sync(0xffffffffu, total, 2);
      const int r = m * 16 + e * 8 + g;
      if (t == 0) {
        stat[(warp * ROWS + r) * 2] = mx[m][e];
        stat[(warp * ROWS + r) * 2 + 1] = total;
      }
#pragma unroll
      for (int n = 0; n < ND; ++n)
        *reinterpret_cast<float2*>(&area[(warp * ROWS + r) * OP + n * 8 + 2 * t]) =
            make_float2(o[m][n][e * 2], o[m][n][e * 2 + 1]);
    }
  }
  if (a.ranks > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else
    __syncthreads();

  // the ranks share the (row, 2 columns) pairs; each joins every warp of
  // every rank, in order
  const uint32_t area_s = wd_smem(area), stat_s = wd_smem(stat);
  const int pairs = a.dim / 2, total = rows * pairs;
  for (int i = rank * (WARPS * 32) + threadIdx.x; i < total; i += a.ranks * (WARPS * 32)) {
    const int r = i / pairs, d = (i - r * pairs) * 2;
    float M = -INFINITY, S = 0.0f, x = 0.0f, y = 0.0f;
    for (int c = 0; c < a.ranks; ++c) {
      uint32_t area_c = area_s, stat_c = stat_s;
      if (a.ranks > 1) {
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(area_c) : "r"(area_s), "r"(c));
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(stat_c) : "r"(stat_s), "r"(c));
      }
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        float2 ms, v;
        asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];"
                     : "=f"(ms.x), "=f"(ms.y) : "r"(stat_c + 8u * (uint32_t)(w * ROWS + r)));
        asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];"
                     : "=f"(v.x), "=f"(v.y) : "r"(area_c + 4u * (uint32_t)((w * ROWS + r) * OP + d)));
        if (ms.x == -INFINITY && ms.y == 0.0f) continue;         // saw no key
        const float mn = fmaxf(M, ms.x);
        const float f0 = fast_exp2(M - mn), f1 = fast_exp2(ms.x - mn);
        S = S * f0 + ms.y * f1;
        x = x * f0 + v.x * f1;
        y = y * f0 + v.y * f1;
        M = mn;
      }
    }
    if (a.parts == 1) {
      const float inv = S == 0.0f ? 0.0f : 1.0f / S;
      const int q = r / a.per, hd = h * a.per + r % a.per;
      OT* dst = static_cast<OT*>(a.out) +
                (((long long)b * a.nq + q) * (a.kv_heads * a.per) + hd) * a.dim + d;
      Slot<OT, 2> so;
      const float f[2] = {x * inv, y * inv};
      pack_slot<OT, 2>(so, f);
      *reinterpret_cast<Slot<OT, 2>*>(dst) = so;
    } else {
      float* dst = a.part + (((long long)item * a.parts + part) * rows + r) * (a.dim + 2);
      *reinterpret_cast<float2*>(dst + d) = make_float2(x, y);
      if (d == 0) *reinterpret_cast<float2*>(dst + a.dim) = make_float2(M, S);
    }
  }
  if (a.ranks > 1)                                   // peers may still read this CTA's rows
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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
