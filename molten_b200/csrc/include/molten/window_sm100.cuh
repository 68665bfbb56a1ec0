// Attention over a sliding window and the first keys, many query rows
// (prompts and chunks), on tcgen05:
//
//   query i of request b stands at p = len_b - nq + i and sees key j iff
//   j <= p and (j > p - window or j < sinks);  o = softmax(q k^T scale) v
//   over the keys it sees, 0 if it sees none.
//
// A work item is a key head of a request and two Q tiles of up to 128 rows;
// a row is (position, head that shares the key head), so grouped heads fill a
// tile with fewer positions and the window's edges cost fewer masked
// products.  The item's key tiles of 128 are those that some row sees: the
// sinks' and the window's.  Each Q tile has its own S and O in TMEM (S0, S1,
// O0, O1: 512 columns at head dim 128), P over S:
//
//   warp 0       TMA: the Q tiles, then K and V tiles through one ring;
//   warp 1       TMEM owner, MMA issuer: S = Q K^T (both operands in shared
//                memory), O += P V with P as the TMEM operand; the two Q tiles
//                alternate, so one's products run under the other's softmax;
//   warps 2, 3   clean the V tiles that not every row sees all of (below);
//   warps 4..7   softmax of Q tile 0 (a thread owns a row), warps 8..11 of
//                tile 1: S from TMEM, running maximum and sum in fp32, P
//                rounded to the type of V (the tensor core takes operands of
//                one type; within 2^-8 or 2^-11 of a weight) back to TMEM.
//
// A 128 x 128 tile takes some 1024 cycles of the tensor core (4 D operations a
// visible pair) and as many of the EX2 unit; what bounds it is the chain of one
// Q tile: S, the exponentials of its halves, P V.  P is handed over by halves,
// so the first half's P V runs under the second's exponentials, and a logit is
// read once: weights are taken from an offset that moves, with O and the sum
// rescaled, only when a logit exceeds it by more than 2^8, so there is no pass
// for the maximum first.  The weights stay below 2^8 and O and the sum share the
// factor, so nothing is lost.  (fp16 weights are taken times 2^7.)
//
// Measured: 8192 tokens, 32 heads over 8, head dim 128, window 2048: 256 us (941
// TFLOP/s of visible pairs), 288 (837) at the clock that seconds of such calls
// leave; 4 x 500 tokens over up to 2900, head dim 64, window 1000: 27.1 us.  With a whole row of S in registers (spills) the first took 489,
// with its maximum first 314.  S by halves, so that it can be computed ahead:
// 270 (N = 64 takes the tensor core as long as N = 128); an issuing warp for
// each Q tile: 310; 4 of 32 exponentials on the FMA pipe: 274 where none was 271;
// two softmax threads a row (16 warps of 96 registers, spills): 387; the next
// half's S loaded ahead: 267.  The waits for S and P poll (all asleep: 270; all
// polling without a pause: 293), the others, of warps with time, sleep.
//
// Where items are fewer than SMs, several CTAs share the key tiles of one; a
// second kernel joins their sums (1 x 64 tokens over 8000, window 4096: 69 -> 36
// us; 1 x 128 over 30000: 425 -> 74).
//
// P = 0 times an infinity or NaN is NaN, so V rows that no query of the item
// sees (behind the length, before the window) are zeroed in shared memory
// before their MMA, and so are infinities and NaN in rows that only some
// queries see; an item that had one of those adds it, from global memory, to
// the outputs of the rows that do see it.
//
// Every mbarrier wait is bounded; on timeout the CTA sets a status bit, stops,
// drains its copies, frees TMEM and returns.
#pragma once

#include "molten/attn_sm100.cuh"

namespace molten {

struct alignas(64) WindowTcArgs {
  CUtensorMap tmap_q;              // q [batch, nq, heads, dim], box {64, per, positions, 1}
  CUtensorMap tmap_k;              // k [batch, cache, kv_heads, dim], box {64, 1, 128, 1}
  CUtensorMap tmap_v;
  const void* v;
  const int* lengths;              // [batch] valid keys, or null: cache
  void* out;                       // [batch, nq, heads, dim] contiguous
  int* status;
  long long v_b, v_s, v_h;         // strides of v in elements
  int batch, nq, cache, kv_heads, per, dim;
  int window, sinks;               // window < 0: every earlier key
  float scale_log2;                // scale * log2(e), positive
  int positions;                   // positions of one Q tile
  int blocks;                      // pairs of Q tiles of a request
  int parts;                       // CTAs that share the key tiles of an item
  float* part;                     // parts > 1: [item][Q tile][128 rows][dim sums, offset, sum of weights, 2 unused]
};

enum WindowTcStatus { kWindowTimeout = 2048 };

// DP: dim padded to 64 or 128.
template <int DP_, int STAGES_>
struct WindowTcLayout {
  static constexpr int DP = DP_, STAGES = STAGES_, DCH = DP / 64, BN = 128;
  static constexpr int CHUNK = 128 * 128;            // 128 rows of 128 bytes
  static constexpr int Q_BYTES = DCH * CHUNK;        // one Q tile
  static constexpr int STAGE_BYTES = DCH * CHUNK;    // one K or V tile
  static constexpr int RING_OFFSET = 2 * Q_BYTES;
  static constexpr int BAR_OFFSET = RING_OFFSET + STAGES * STAGE_BYTES;
  // full[S] empty[S] clean[S] q_full[2] q_empty[2] s_full[2] p_full[4] o_half[2] o_full[2] o_free[2] done
  static constexpr int NUM_BARS = 3 * STAGES + 17;
  static constexpr int SMEM_BYTES = BAR_OFFSET + NUM_BARS * 8 + 8 + 8 * 4 + 8 + 1024;
  static constexpr int THREADS = 384;
  static constexpr uint32_t TM_S = 0, TM_O = 256;    // + 128 for Q tile 1
};

template <class L> struct WindowTcBars {
  uint32_t base;
  __device__ __forceinline__ uint32_t full(int i) const { return base + 8u * i; }
  __device__ __forceinline__ uint32_t empty(int i) const { return base + 8u * (L::STAGES + i); }
  __device__ __forceinline__ uint32_t clean(int i) const { return base + 8u * (2 * L::STAGES + i); }
  __device__ __forceinline__ uint32_t q_full(int t) const { return base + 8u * (3 * L::STAGES + t); }
  __device__ __forceinline__ uint32_t q_empty(int t) const { return base + 8u * (3 * L::STAGES + 2 + t); }
  __device__ __forceinline__ uint32_t s_full(int t) const { return base + 8u * (3 * L::STAGES + 4 + t); }
  __device__ __forceinline__ uint32_t p_full(int t, int half) const { return base + 8u * (3 * L::STAGES + 13 + 2 * t + half); }
  __device__ __forceinline__ uint32_t o_half(int t) const { return base + 8u * (3 * L::STAGES + 6 + t); }
  __device__ __forceinline__ uint32_t o_full(int t) const { return base + 8u * (3 * L::STAGES + 8 + t); }
  __device__ __forceinline__ uint32_t o_free(int t) const { return base + 8u * (3 * L::STAGES + 10 + t); }
  __device__ __forceinline__ uint32_t done() const { return base + 8u * (3 * L::STAGES + 12); }
};

struct WindowTcShared {
  uint8_t* q;                      // 1024-aligned
  uint8_t* ring;
  uint32_t bars;
  uint32_t* tmem_slot;
  volatile int* abort_flag;
  int* dirty;                      // [8] by item number: the latest item + 1 with cleaned infinities or NaN
};

template <class L>
__device__ __forceinline__ WindowTcShared window_tc_carve(uint8_t* raw) {
  WindowTcShared s;
  const uintptr_t base = (reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023);
  s.q = reinterpret_cast<uint8_t*>(base);
  s.ring = s.q + L::RING_OFFSET;
  s.bars = smem_u32(s.q + L::BAR_OFFSET);
  s.tmem_slot = reinterpret_cast<uint32_t*>(s.q + L::BAR_OFFSET + L::NUM_BARS * 8);
  s.abort_flag = reinterpret_cast<volatile int*>(s.tmem_slot + 1);
  s.dirty = reinterpret_cast<int*>(s.tmem_slot + 2);
  return s;
}

__device__ __forceinline__ void window_tc_fail(const WindowTcShared& s, const WindowTcArgs& args) {
  *s.abort_flag = 1;
  if (args.status) atomicOr(args.status, kWindowTimeout);
}

// The key tiles of a work item: [0, sink) and [start, end) in ascending order;
// of these Q tile t needs those below need_sink[t] and in [lo[t], hi[t]).
// PARTS: items are shared by args.parts CTAs, each with a run of the tiles.
template <bool PARTS>
struct WindowItem {
  int b, h, first, len;            // first: position of query 0
  int i0;                          // first query of the item
  int sink, start, end, tiles, skip;   // skip: tiles of the parts before
  int lo[2], hi[2], need_sink[2];
  int pa[2], pb[2];                // positions of the Q tiles' first and last rows; pb < pa: none
  __device__ __forceinline__ WindowItem(const WindowTcArgs& a, int item) {
    const int part = PARTS ? item % a.parts : 0, whole_item = PARTS ? item / a.parts : item;
    const int block = whole_item % a.blocks, rest = whole_item / a.blocks;
    h = rest % a.kv_heads;
    b = rest / a.kv_heads;
    int n = a.lengths ? a.lengths[b] : a.cache;
    n = n < 0 ? 0 : (n > a.cache ? a.cache : n);
    len = n;
    first = n - a.nq;
    i0 = block * 2 * a.positions;
    start = 0x7fffffff;
    end = 0;
    sink = 0x7fffffff;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int ia = i0 + t * a.positions, ib = min(ia + a.positions, a.nq) - 1;
      pa[t] = max(first + ia, 0);                    // rows before the first key see nothing
      pb[t] = first + ib;
      if (ib < ia || pb[t] < 0) {
        pa[t] = 0; pb[t] = -1; lo[t] = 0; hi[t] = 0; need_sink[t] = 0;
        continue;
      }
      lo[t] = (a.window < 0 || pa[t] < a.window ? 0 : pa[t] - a.window + 1) / 128;
      hi[t] = pb[t] / 128 + 1;
      need_sink[t] = min((a.sinks + 127) / 128, hi[t]);
      start = min(start, lo[t]);
      end = max(end, hi[t]);
      sink = min(sink, min(need_sink[t], lo[t]));
    }
    // (a later Q tile's sinks may reach past the earlier one's window start:
    // they are inside [start, end) then)
    if (end == 0) { sink = 0; start = 0; }
    else if (pb[0] >= pa[0] && pb[1] >= pa[1]) sink = min(max(need_sink[0], need_sink[1]), start);
    else sink = min(sink, start);
    tiles = sink + end - start;
    skip = 0;
    if constexpr (PARTS) {
      skip = (int)((long long)tiles * part / a.parts);
      tiles = (int)((long long)tiles * (part + 1) / a.parts) - skip;
    }
  }
  __device__ __forceinline__ int tile(int u) const {
    const int v = PARTS ? u + skip : u;
    return v < sink ? v : v - sink + start;
  }
  // (selects, not an index: the members stay in registers where t is a variable)
  static __device__ __forceinline__ int of(const int (&x)[2], int t) { return t == 0 ? x[0] : x[1]; }
  __device__ __forceinline__ bool any(int t) const { return of(pb, t) >= of(pa, t); }
  // (tiles ascend: some tile of this part is among the sinks' or the window's)
  __device__ __forceinline__ bool has(int t) const {
    if (!PARTS || !any(t)) return any(t);
    if (tiles == 0) return false;
    const int j0 = tile(0), j1 = tile(tiles - 1);
    return j0 < of(need_sink, t) ||
           max(max(j0, start), of(lo, t)) <= min(j1, of(hi, t) - 1);
  }
  __device__ __forceinline__ bool need(int t, int j) const {
    return any(t) && (j < of(need_sink, t) || (j >= of(lo, t) && j < of(hi, t)));
  }
  // every row of Q tile t sees all of key tile j
  __device__ __forceinline__ bool whole(const WindowTcArgs& a, int t, int j) const {
    const int k = j * 128;
    return k + 127 <= of(pa, t) && first + i0 + t * a.positions >= 0 &&
           (a.window < 0 || k > of(pb, t) - a.window || k + 128 <= a.sinks);
  }
  // V needs no cleaning: whole for each Q tile that needs it, and both do
  __device__ __forceinline__ bool clean(const WindowTcArgs& a, int j) const {
    return (!need(0, j) || whole(a, 0, j)) && (!need(1, j) || whole(a, 1, j));
  }
};

// The positions of the rows are one run from pa to pb, so the keys some row
// sees are one run (and the sinks).
__device__ __forceinline__ bool window_tc_any(const WindowTcArgs& a, int pa, int pb, int j) {
  return j <= pb && (a.window < 0 || j > pa - a.window || j < a.sinks);
}
// The lowest n bits.
__device__ __forceinline__ uint32_t window_tc_bits(int n) {
  return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u;
}
__device__ __forceinline__ bool window_tc_sees(const WindowTcArgs& a, int p, int j) {
  return j <= p && (a.window < 0 || j > p - a.window || j < a.sinks);
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
               " [%0], [%1, {%3, %4, %5, %6}], [%2];"
               :: "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// D (+)= A B with A in TMEM (two 16-bit values a column)
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\t"
               "setp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               :: "r"(d_tmem), "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* u) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {"
               "%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
               "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32"
               "};"
               :: "r"(taddr),
                 "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]),
                 "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]),
                 "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]),
                 "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31]) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&u)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]),
        "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// One lane of a converged warp, the same at each call.
__device__ __forceinline__ bool window_tc_elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0u;
}

template <class L>
__device__ __forceinline__ void window_tc_init(const WindowTcShared& s, const WindowTcArgs& args) {
  const int tid = threadIdx.x, warp = tid / 32;
  if (tid == 0) {
    const WindowTcBars<L> b{s.bars};
    for (int i = 0; i < L::STAGES; ++i) {
      mbar_init(b.full(i), 1);
      mbar_init(b.empty(i), 1);
      mbar_init(b.clean(i), 2);                      // the two cleaning warps
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(b.q_full(t), 1);
      mbar_init(b.q_empty(t), 1);
      mbar_init(b.s_full(t), 1);
      mbar_init(b.p_full(t, 0), 4);                  // the Q tile's softmax warps
      mbar_init(b.p_full(t, 1), 4);
      mbar_init(b.o_half(t), 1);
      mbar_init(b.o_full(t), 1);
      mbar_init(b.o_free(t), 4);
    }
    mbar_init(b.done(), 1);
    *s.abort_flag = 0;
    for (int i = 0; i < 8; ++i) s.dirty[i] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" :: "l"(&args.tmap_q) : "memory");
    asm volatile("prefetch.tensormap [%0];" :: "l"(&args.tmap_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" :: "l"(&args.tmap_v) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_u32(s.tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
}

// Infinities and NaN of V that were cleaned away, added to the stored output
// row of position p from the keys it sees (any weight above 0 carries them into
// the sum).
template <bool PARTS, typename T, typename OT>
__device__ __noinline__ void window_tc_add_dirty(const WindowTcArgs& args, int item, int p, OT* dst) {
  const WindowItem<PARTS> w(args, item);
#pragma unroll 1
  for (int u = 0; u < w.tiles; ++u) {
    const int j = w.tile(u);
    if (w.clean(args, j)) continue;
#pragma unroll 1
    for (int key = j * 128; key < j * 128 + 128 && key < w.len; ++key) {
      if (!window_tc_sees(args, p, key)) continue;
      const T* v = static_cast<const T*>(args.v) + w.b * args.v_b + key * args.v_s + w.h * args.v_h;
#pragma unroll 1
      for (int c = 0; c < args.dim; ++c) {
        const float x = to_f32(v[c]);
        if (!isfinite(x)) dst[c] = from_f32<OT>(to_f32(dst[c]) + x);
      }
    }
  }
}

// sum + 0 x, for two 16-bit numbers: 0, or NaN from the first infinity or NaN on.
template <typename T>
__device__ __forceinline__ uint32_t window_tc_zeros(uint32_t x, uint32_t sum) {
  if constexpr (std::is_same<T, f16>::value)
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(sum) : "r"(x), "r"(0u), "r"(sum));
  else
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(sum) : "r"(x), "r"(0u), "r"(sum));
  return sum;
}

template <class L, typename T, typename OT, bool PARTS>
__device__ __forceinline__ void window_tc_roles(const WindowTcShared& s, const WindowTcArgs& args) {
  constexpr bool F16IN = std::is_same<T, f16>::value;
  constexpr uint32_t S = L::STAGES;
  tc_fence_after();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t tmem = *s.tmem_slot;
  const WindowTcBars<L> bar{s.bars};
  const int items = args.batch * args.kv_heads * args.blocks * (PARTS ? args.parts : 1);
  // ring entries in order K, V, K, V ...: entry e lies in stage e % S, and the
  // barriers of its e / S-th use have that parity; V tile e / 2 is passed on by
  // the cleaning warps through barrier clean(e / 2 % S)
  bool ok = true;
  auto wait = [&](uint32_t b, uint32_t parity) {
    if (!attn_wait(b, parity & 1u)) { window_tc_fail(s, args); ok = false; }
    return ok;
  };

  if (warp == 0) {
    // ------------------------------------------------------- TMA producer
    if (lane == 0) {
      const uint32_t q_bytes = (uint32_t)(L::DCH * 128 * args.per * args.positions);
      uint32_t entry = 0, qn[2] = {0, 0};
      auto load = [&](const CUtensorMap* map, const WindowItem<PARTS>& w, int j) {
        const uint32_t st = entry % S;
        if (!wait(bar.empty(st), entry / S + 1u)) return;
        mbar_expect_tx(bar.full(st), (uint32_t)L::STAGE_BYTES);
#pragma unroll
        for (int c = 0; c < L::DCH; ++c)
          tma_load_4d(smem_u32(s.ring + st * L::STAGE_BYTES + c * L::CHUNK), map, bar.full(st),
                      c * 64, w.h, j * 128, w.b);
        ++entry;
      };
      for (int it = blockIdx.x; it < items && ok; it += gridDim.x) {
        const WindowItem<PARTS> w(args, it);
        for (int t = 0; t < 2; ++t) {
          if (!w.has(t)) continue;
          if (!wait(bar.q_empty(t), qn[t] + 1u)) break;
          ++qn[t];
          mbar_expect_tx(bar.q_full(t), q_bytes);
#pragma unroll
          for (int c = 0; c < L::DCH; ++c)
            tma_load_4d(smem_u32(s.q + t * L::Q_BYTES + c * L::CHUNK), &args.tmap_q, bar.q_full(t),
                        c * 64, w.h * args.per, w.i0 + t * args.positions, w.b);
        }
        for (int u = 0; u < w.tiles && ok; ++u) {
          load(&args.tmap_k, w, w.tile(u));
          if (ok) load(&args.tmap_v, w, w.tile(u));
        }
      }
      if (!ok) {
        // let the copies this thread issued land before the CTA can exit
        bool landed = true;
        for (uint32_t i = 0; i < S && i < entry; ++i) {
          const uint32_t e = entry - 1u - i;
          landed &= attn_wait(bar.full(e % S), (e / S) & 1u);
        }
        for (int t = 0; t < 2; ++t)
          if (qn[t]) landed &= attn_wait(bar.q_full(t), (qn[t] + 1u) & 1u);
        if (!landed && args.status) atomicOr(args.status, kWindowTimeout);
      }
    }
  } else if (warp == 1) {
    // --------------------------------------------------------- MMA issuer
    // (the whole warp takes these steps, so that what describes an MMA is the
    // same in every lane and held in uniform registers; one lane issues.  With
    // the steps in one lane only, each MMA took as long to issue as to run)
    {
      const bool leader = window_tc_elect();
      auto wait_all = [&](uint32_t b, uint32_t parity) {
        ok = __all_sync(0xffffffffu, mbar_wait(b, parity & 1u));
        if (!ok && lane == 0) window_tc_fail(s, args);
        return ok;
      };
      constexpr uint32_t IDESC_S = umma_idesc<128, 128, F16IN, true>();
      constexpr uint32_t IDESC_O = umma_idesc<128, L::DP, F16IN, false>();
      uint32_t qn[2] = {0, 0}, pn[2] = {0, 0}, on[2] = {0, 0};   // Q tiles, P tiles, items of O
      // the next ring entry and the next V's cleaning barrier, with their parities
      uint32_t st = 0, ph = 0, cst = 0, cph = 0;
      auto advance = [](uint32_t& at, uint32_t& parity) {
        if (++at == S) { at = 0; parity ^= 1u; }
      };
      // descriptors without their address (it is added in units of 16 bytes)
      const uint64_t by_row = umma_desc(0u, 16u, 1024u), by_col = umma_desc(0u, (uint32_t)L::CHUNK, 1024u);
      const uint32_t q_at = smem_u32(s.q) >> 4, ring_at = smem_u32(s.ring) >> 4;
      for (int it = blockIdx.x; it < items && ok; it += gridDim.x) {
        const WindowItem<PARTS> w(args, it);
        bool begun[2] = {false, false}, asked[2] = {false, false};   // O_t holds sums; Q_t is there
        bool needed[2] = {false, false};             // by Q tile t: the key tile before
        // step u: P V of tile u - 1 and S of tile u, for either Q tile in turn
        for (int u = 0; u <= w.tiles && w.tiles > 0 && ok; ++u) {
          const bool has_k = u < w.tiles, has_v = u > 0;
          const int j = has_k ? w.tile(u) : 0;
          uint32_t v_st = 0, k_st = 0;
          if (has_v) {
            if (!wait_all(bar.clean(cst), cph)) break;   // (the cleaning warps have waited for the tile)
            v_st = st;
            advance(st, ph);
            advance(cst, cph);
          }
          if (has_k) {
            if (!wait_all(bar.full(st), ph)) break;
            k_st = st;
            advance(st, ph);
          }
          const uint64_t v_desc = by_col + (ring_at + v_st * (uint32_t)(L::STAGE_BYTES / 16));
          const uint64_t k_desc = by_row + (ring_at + k_st * (uint32_t)(L::STAGE_BYTES / 16));
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (has_v && needed[t]) {
              if (!begun[t] && !wait_all(bar.o_free(t), on[t]++ + 1u)) break;
              const uint32_t d = tmem + L::TM_O + 128u * t, p = tmem + L::TM_S + 128u * t;
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                if (!wait_all(bar.p_full(t, half), pn[t])) break;
                tc_fence_after();
                if (leader) {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                  umma_f16_ts(d, p + 64u * half + 8u * kk, v_desc + 128u * (4 * half + kk), IDESC_O,
                              begun[t] || (half | kk) != 0 ? 1u : 0u);
                if (half == 0) umma_commit(bar.o_half(t));
                }
              }
              if (!ok) break;
              ++pn[t];
              begun[t] = true;
            }
            needed[t] = has_k && w.need(t, j);
            if (needed[t]) {
              // (S_t is free: its last P has been used, and MMAs run in order)
              if (!asked[t]) {
                if (!wait_all(bar.q_full(t), qn[t]++)) break;
                asked[t] = true;
              }
              tc_fence_after();
              const uint32_t d = tmem + L::TM_S + 128u * t;
              const uint64_t q_desc = by_row + (q_at + t * (uint32_t)(L::Q_BYTES / 16));
              if (leader) {
#pragma unroll
              for (int c = 0; c < L::DCH; ++c)
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                  umma_f16(d, q_desc + (uint32_t)(c * (L::CHUNK / 16) + 2 * kk),
                           k_desc + (uint32_t)(c * (L::CHUNK / 16) + 2 * kk), IDESC_S, (c | kk) != 0 ? 1u : 0u);
              umma_commit(bar.s_full(t));
              }
            }
          }
          if (!ok) break;
          if (leader) {
            if (has_v) umma_commit(bar.empty(v_st));
            if (has_k) umma_commit(bar.empty(k_st));
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (u == w.tiles - 1 && asked[t]) umma_commit(bar.q_empty(t));     // the item's last S
              if (u == w.tiles && begun[t]) umma_commit(bar.o_full(t));          // its last P V
            }
          }
          __syncwarp();
        }
      }
      // all MMAs this thread issued must finish before TMEM is released
      if (leader) {
        umma_commit(bar.done());
        if (!attn_wait(bar.done(), 0u)) { if (args.status) atomicOr(args.status, kWindowTimeout); }
      }
    }
  } else if (warp < 4) {
    // ----------------------------------------------------------- cleaning
    // (every V tile is seen and passed on, so that the parities of a stage's
    // barriers cannot run ahead of these warps)
    uint32_t n = 0, seq = 0;
    for (int it = blockIdx.x; it < items && ok; it += gridDim.x, ++seq) {
      const WindowItem<PARTS> w(args, it);
      const bool v0 = w.pb[0] >= w.pa[0], v1 = w.pb[1] >= w.pa[1];
      const int pa = v0 ? w.pa[0] : w.pa[1], pb = v1 ? w.pb[1] : w.pb[0];
      for (int u = 0; u < w.tiles && ok; ++u) {
        const int j = w.tile(u);
        const uint32_t e = 2u * (n + u) + 1u;
        const bool got = attn_wait(bar.full(e % S), (e / S) & 1u);
        if (!__all_sync(0xffffffffu, got && !*s.abort_flag)) {
          if (lane == 0) window_tc_fail(s, args);
          ok = false;
          break;
        }
        bool found = false;
#pragma unroll 1
        for (int r = (warp - 2) * 32 + lane; r < 128 && !w.clean(args, j); r += 64) {
          const int key = j * 128 + r;
          const bool any = key < w.len && window_tc_any(args, pa, pb, key);
          const bool all = key <= pa && (args.window < 0 || key > pb - args.window || key < args.sinks);
          if (any && all) continue;
          uint8_t* row = s.ring + (e % S) * L::STAGE_BYTES + r * 128;
          // 16-byte chunks, the lanes' on different banks.  0 x sums up to NaN in a
          // row with an infinity or NaN (rare: those are looked through again)
          auto chunk = [&](int q) {
            return reinterpret_cast<uint4*>(row + (q >> 3) * L::CHUNK + (((q + lane) & 7) << 4));
          };
          uint32_t sum = 0u;
#pragma unroll 8
          for (int q = 0; q < L::DCH * 8; ++q) {
            if (!any) { *chunk(q) = make_uint4(0u, 0u, 0u, 0u); continue; }
            const uint4 x = *chunk(q);
            sum = window_tc_zeros<T>(x.x, window_tc_zeros<T>(x.y, window_tc_zeros<T>(x.z, window_tc_zeros<T>(x.w, sum))));
          }
          if ((sum & 0x7FFF7FFFu) == 0u) continue;
          found = true;
#pragma unroll 1
          for (int q = 0; q < L::DCH * 8; ++q) {
            uint4 x = *chunk(q);
            uint32_t* xs = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              constexpr uint32_t EXP = F16IN ? 0x7C00u : 0x7F80u;
              if ((xs[i] & EXP) == EXP) xs[i] &= 0xFFFF0000u;
              if ((xs[i] >> 16 & EXP) == EXP) xs[i] &= 0x0000FFFFu;
            }
            *chunk(q) = x;
          }
        }
        // (numbers only grow: the cleaning warps may be any number of items ahead of
        // the softmax, since items without key tiles take no stage of the ring)
        if (found) atomicMax(&s.dirty[seq & 7u], (int)seq + 1);
        // the writes come before the tensor core's reads
        fence_async_shared();
        __threadfence_block();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar.clean(e / 2u % S));
      }
      n += (uint32_t)w.tiles;
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int t = (warp - 4) / 4, quarter = warp % 4;
    const int r = quarter * 32 + lane;               // row of the Q tile = TMEM lane
    const uint32_t lane_at = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_at = tmem + lane_at + L::TM_S + 128u * t;
    const uint32_t o_at = tmem + lane_at + L::TM_O + 128u * t;
    const float C2 = args.scale_log2;
    // the largest weight lies between 2^LIFT and 2^(LIFT + 8): 8 bits of growth of
    // the maximum are left in the weights.  fp16 ends at 2^16 and keeps all its bits
    // down to 2^-14 and none below 2^-25, so its weights are lifted (by 11 with 4 bits
    // of growth: 4 x 500 tokens took 5% longer)
    constexpr float LIFT = F16IN ? 7.0f : 0.0f;
    const float slack = 8.0f / C2;
    uint32_t sn = 0, rn = 0, seq = 0;                // tiles of S; items with any
    for (int it = blockIdx.x; it < items && ok; it += gridDim.x, ++seq) {
      const WindowItem<PARTS> w(args, it);
      const int i = w.i0 + t * args.positions + r / args.per;    // this row's query
      const bool real = r < args.per * args.positions && i < args.nq;
      const int p = w.first + i;
      // weights are 2^(x C2 + off); a logit above `limit` moves `off`
      float off = 0.0f, limit = -INFINITY, sum = 0.0f;
      const bool run = w.has(t);
      if (run) {
        bool begun = false;
        for (int u = 0; u < w.tiles; ++u) {
          const int j = w.tile(u);
          if (!w.need(t, j)) continue;
          const bool whole = w.whole(args, t, j);
          // columns behind c0 (or before cs) and up to c1 are seen
          const int c1 = p - j * 128 + 1;
          const int c0 = args.window < 0 ? 0 : p - args.window - j * 128 + 1;
          const int cs = args.sinks - j * 128;
          const bool got = mbar_wait(bar.s_full(t), sn & 1u);
          if (!__all_sync(0xffffffffu, got && !*s.abort_flag)) {
            if (lane == 0) window_tc_fail(s, args);
            ok = false;
            break;
          }
          ++sn;
          tc_fence_after();
          // 64 columns of S at a time, each read once: half a row leaves registers
          // for the rest (a whole one spilled, at twice the time), and its P V
          // runs under the other half's exponentials
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            float x[64];
            tmem_ld64(s_at + 64 * half, x);
            if (!whole) {
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const int k = 64 * half + 32 * q;
                const uint32_t seen = window_tc_bits(c1 - k) & (~window_tc_bits(c0 - k) | window_tc_bits(cs - k));
#pragma unroll
                for (int c = 0; c < 32; ++c)
                  if (!(seen >> c & 1u)) x[32 * q + c] = -INFINITY;
              }
            }
            float top[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) top[q] = fmaxf(x[q], x[q + 4]);
#pragma unroll
            for (int c = 8; c < 64; c += 8)
#pragma unroll
              for (int q = 0; q < 4; ++q) top[q] = fmaxf(fmaxf(top[q], x[c + q]), x[c + 4 + q]);
            const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            // (each row by its own maximum: no row's result depends on another's)
            const bool grown = real && mx > limit;
            if (__any_sync(0xffffffffu, grown)) {
              const float moved = grown ? LIFT - mx * C2 : off;
              // (the first maximum of a row: O and the sum are 0)
              const float fix = grown && limit > -INFINITY ? fast_exp2(moved - off) : 1.0f;
              off = moved;
              limit = grown ? mx + slack : limit;
              sum *= fix;
              // P V of all tiles before is done (their S came first); of this one's
              // first half it may be running
              if (half == 1) {
                const bool done = attn_wait(bar.o_half(t), (sn + 1u) & 1u);      // (tile sn - 1)
                if (!__all_sync(0xffffffffu, done ? 1 : 0)) {
                  if (lane == 0) window_tc_fail(s, args);
                  ok = false;
                  break;
                }
                tc_fence_after();
              }
              if (begun || half == 1) {
#pragma unroll 1
                for (int c = 0; c < L::DP; c += 32) {
                  float o[32];
                  tmem_ld32(o_at + c, o);
                  uint32_t y[32];
#pragma unroll
                  for (int q = 0; q < 32; ++q) y[q] = __float_as_uint(o[q] * fix);
                  tmem_st32(o_at + c, y);
                }
              }
            }
            const float2 scale2 = make_float2(C2, C2), off2 = make_float2(off, off);
            float2 part[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
            uint32_t y[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              float2 e = ffma2(make_float2(x[2 * c], x[2 * c + 1]), scale2, off2);
              e.x = fast_exp2(e.x);
              e.y = fast_exp2(e.y);
              part[c % 2] = fadd2(part[c % 2], e);
              Slot<T, 2> two;
              const float f[2] = {e.x, e.y};
              pack_slot<T, 2>(two, f);
              y[c] = *reinterpret_cast<const uint32_t*>(&two);
            }
            tmem_st32(s_at + 64 * half, y);          // (each half's P over its own S)
            sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar.p_full(t, half));
          }
          if (!ok) break;
          begun = true;
        }
        if (!ok) break;
        const bool done = attn_wait(bar.o_full(t), rn++ & 1u);
        if (!__all_sync(0xffffffffu, done && !*s.abort_flag)) {
          if (lane == 0) window_tc_fail(s, args);
          ok = false;
          break;
        }
        tc_fence_after();
      }
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      // (a later item's number says nothing of this one: it is looked through)
      const bool dirty = *(volatile int*)&s.dirty[seq & 7u] > (int)seq;
      if constexpr (PARTS) {
        // this part's sums as they are, with their offset (+inf: no key seen)
        float* mine = args.part + ((long long)(it * 2 + t) * 128 + r) * (args.dim + 4);
#pragma unroll 1
        for (int c = 0; c < L::DP; c += 16) {
          uint32_t o[16];
          if (run) tmem_ld16(o_at + c, o);
          if (!real || !run || c >= args.dim) continue;
#pragma unroll
          for (int q = 0; q < 16; q += 4)
            if (c + q < args.dim)
              *reinterpret_cast<uint4*>(mine + c + q) = make_uint4(o[q], o[q + 1], o[q + 2], o[q + 3]);
        }
        if (real) {
          *reinterpret_cast<float2*>(mine + args.dim) =
              limit == -INFINITY && sum == 0.0f ? make_float2(INFINITY, 0.0f) : make_float2(off, sum);
          if (dirty && run) window_tc_add_dirty<PARTS, T, float>(args, it, p, mine);
        }
        if (run) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar.o_free(t));
        }
        continue;
      }
      OT* dst = static_cast<OT*>(args.out) +
                (((long long)w.b * args.nq + i) * args.kv_heads * args.per + w.h * args.per + r % args.per) *
                    (long long)args.dim;
      // 16 columns at a time, whole sectors where rows start on one (each lane
      // writes its own row)
      constexpr int WORDS = 4 * (int)sizeof(OT);     // of 16 values
      const bool wide = args.dim % 16 == 0 && (reinterpret_cast<uintptr_t>(args.out) & 31u) == 0u;
#pragma unroll 1
      for (int c = 0; c < L::DP; c += 32) {
        float o[32];
        if (run) tmem_ld32(o_at + c, o);             // (the whole warp)
        if (c >= args.dim) continue;
        uint32_t y[2 * WORDS];
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const float f[2] = {sum == 0.0f ? 0.0f : o[2 * q] * inv, sum == 0.0f ? 0.0f : o[2 * q + 1] * inv};
          if constexpr (sizeof(OT) == 4) {
            y[2 * q] = __float_as_uint(f[0]);
            y[2 * q + 1] = __float_as_uint(f[1]);
          } else {
            Slot<OT, 2> two;
            pack_slot<OT, 2>(two, f);
            y[q] = *reinterpret_cast<const uint32_t*>(&two);
          }
        }
        if (!real) continue;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          if (c + 16 * q >= args.dim) break;
          uint32_t* at = reinterpret_cast<uint32_t*>(dst + c + 16 * q);
          const uint32_t* v = y + WORDS * q;
          if (wide) {
#pragma unroll
            for (int k = 0; k < WORDS; k += 8)
              asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                           :: "l"(at + k), "r"(v[k]), "r"(v[k + 1]), "r"(v[k + 2]), "r"(v[k + 3]), "r"(v[k + 4]),
                              "r"(v[k + 5]), "r"(v[k + 6]), "r"(v[k + 7]) : "memory");
          } else {
            // (dim is a multiple of 8 columns)
            const int words = c + 16 * q + 8 < args.dim ? WORDS : WORDS / 2;
#pragma unroll
            for (int k = 0; k < WORDS; k += 4)
              if (k < words) *reinterpret_cast<uint4*>(at + k) = make_uint4(v[k], v[k + 1], v[k + 2], v[k + 3]);
          }
        }
      }
      if (dirty && real) window_tc_add_dirty<PARTS, T, OT>(args, it, p, dst);
      if (run) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar.o_free(t));
      }
    }
  }
}

// The parts of each row joined: a warp to a row of a Q tile.  With o_p the sums
// under offset off_p, o = sum_p o_p 2^(off - off_p) for off = min off_p.
template <typename OT>
__device__ __forceinline__ void window_tc_join(const WindowTcArgs& args) {
  const int lane = threadIdx.x % 32, pitch = args.dim + 4;
  const long long id = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  const int r = (int)(id % 128), t = (int)(id / 128 % 2);
  const long long item = id / 256;                   // without the part
  if (item >= (long long)args.batch * args.kv_heads * args.blocks) return;
  const int block = (int)(item % args.blocks);
  const long long rest = item / args.blocks;
  const int h = (int)(rest % args.kv_heads), b = (int)(rest / args.kv_heads);
  const int i = (block * 2 + t) * args.positions + r / args.per;
  if (r >= args.per * args.positions || i >= args.nq) return;
  const float* mine = args.part + ((item * args.parts * 2 + t) * 128 + r) * (long long)pitch;
  const long long step = 256ll * pitch;              // to the next part
  // a lane to a part: its offset and weight (32 parts at most)
  float2 z = make_float2(INFINITY, 0.0f);
  if (lane < args.parts) z = *reinterpret_cast<const float2*>(mine + lane * step + args.dim);
  float off = z.x, sum;
#pragma unroll
  for (int d = 16; d >= 1; d /= 2) off = fminf(off, __shfl_xor_sync(0xffffffffu, off, d));
  const float f = z.x == INFINITY ? 0.0f : fast_exp2(off - z.x);     // +inf: it saw no key
  sum = z.x == INFINITY ? 0.0f : z.y * f;
#pragma unroll
  for (int d = 16; d >= 1; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int p = 0; p < args.parts; ++p) {
    const float fp = __shfl_sync(0xffffffffu, f, p);
    const bool none = __shfl_sync(0xffffffffu, z.x, p) == INFINITY;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = lane + 32 * q;
      const float x = !none && c < args.dim ? mine[p * step + c] : 0.0f;
      o[q] += isfinite(x) ? x * fp : x;              // (an infinity stays one under any weight)
    }
  }
  OT* dst = static_cast<OT*>(args.out) +
            (((long long)b * args.nq + i) * args.kv_heads * args.per + h * args.per + r % args.per) * args.dim;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int c = lane + 32 * q;
    if (c < args.dim) dst[c] = from_f32<OT>(sum == 0.0f ? 0.0f : o[q] / sum);
  }
}

template <class L>
__device__ __forceinline__ void window_tc_teardown(const WindowTcShared& s) {
  if (threadIdx.x / 32 == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                 :: "r"(*s.tmem_slot), "r"(512u) : "memory");
  }
}

}  // namespace molten
