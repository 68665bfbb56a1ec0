// Rotary embedding with per-token positions on up to four axes.
//
//   pair i of token t turns by the angle of table row pos[axis(i)][t]:
//   (x0, x1) -> (x0 c - x1 s, x0 s + x1 c),  c = cos[row, i], s = sin[row, i]
//
// axis(i) is the section that holds pair i (bound[a] = first pair after
// section a).  Pairs are (i, i + D/2) ("half") or (2i, 2i + 1).  A negative
// position marks padding: those pairs are copied.  A position past the table
// sets kRopePositionRange in the status word, and its pairs are copied too.  (A
// thread whose slot holds such a pair takes a way of its own, so that the other
// keeps its registers: with the choice among the products 4 x 4096 tokens took 60
// us for 51.)
// fp32 arithmetic, one rounding to the output type.
//
// Bound by HBM (x in, x out).  A thread keeps one slot of pairs of one token,
// loads that slot's cos and sin once and turns up to HPT heads with it, all
// their loads issued first: the table costs one read per HPT heads instead of
// one per head (it is fp32 and as wide as x, so it would triple the L1
// traffic).  Every element is read and written by one thread, the reads first, so
// out may be x: x is loaded as memory that changes.
//
// Measured, bf16 with fp32 tables: 4 x 4096 tokens of 32 heads of 128, one axis
// 45.0 us (6.0 TB/s), three axes at random positions 49.6 (each section's table
// rows come from L2); 48 tokens of 40 heads 2.1 us.
#pragma once

#include "molten/common.cuh"

namespace molten {

struct RopePosArgs {
  const void* x;                   // [tokens, heads, dim], strides below, dim contiguous
  const void* cos_t;               // [table_rows, dim/2], or packed [table_rows, dim]
  const void* sin_t;               // [table_rows, dim/2]; unused when packed
  const int* pos;                  // [axes, tokens]
  void* out;                       // [tokens, heads, dim] contiguous
  int* status;
  long long tokens, x_token, x_head, table_rows;
  int heads, dim, axes, head_lanes;
  int bound[4];                    // first pair after each section
  int tokens_per_cta, reserved;
};

enum RopePosStatus { kRopePositionRange = 4096 };

// cos and sin of the NP pairs from p0 on; bit e of the result: pair e stays as it is.
template <typename TT, int NP, bool PACKED, bool TVEC>
__device__ __forceinline__ uint32_t rope_table(const RopePosArgs& a, long long token, int p0,
                                           float (&cs)[NP], float (&sn)[NP]) {
  const int half = a.dim / 2;
  int ax = 0;
  while (ax + 1 < a.axes && p0 >= a.bound[ax]) ++ax;
  const TT* ct = static_cast<const TT*>(a.cos_t);
  const TT* st = static_cast<const TT*>(a.sin_t);
  const bool one_axis = ax + 1 >= a.axes || p0 + NP <= a.bound[ax];
  if (TVEC && one_axis) {
    const long long row = a.pos[(long long)ax * a.tokens + token];
    if (row >= 0 && row < a.table_rows) {
      if constexpr (PACKED) {
        const Slot<TT, 2 * NP> t = load_slot<kLoadDefault, TT, 2 * NP>(ct + row * a.dim + 2 * p0);
#pragma unroll
        for (int e = 0; e < NP; ++e) { cs[e] = to_f32(t.v[2 * e]); sn[e] = to_f32(t.v[2 * e + 1]); }
      } else {
        const Slot<TT, NP> c = load_slot<kLoadDefault, TT, NP>(ct + row * half + p0);
        const Slot<TT, NP> s = load_slot<kLoadDefault, TT, NP>(st + row * half + p0);
#pragma unroll
        for (int e = 0; e < NP; ++e) { cs[e] = to_f32(c.v[e]); sn[e] = to_f32(s.v[e]); }
      }
    } else {
      if (row >= 0 && a.status) atomicOr(a.status, kRopePositionRange);
#pragma unroll
      for (int e = 0; e < NP; ++e) { cs[e] = 1.0f; sn[e] = 0.0f; }
      return (1u << NP) - 1u;
    }
    return 0u;
  }
  uint32_t stay = 0u;
#pragma unroll
  for (int e = 0; e < NP; ++e) {
    const int p = p0 + e;
    while (ax + 1 < a.axes && p >= a.bound[ax]) ++ax;
    const long long row = a.pos[(long long)ax * a.tokens + token];
    const bool in = row >= 0 && row < a.table_rows;
    if (row >= a.table_rows && a.status) atomicOr(a.status, kRopePositionRange);
    stay |= (in ? 0u : 1u) << e;
    if constexpr (PACKED) {
      cs[e] = in ? to_f32(ct[row * a.dim + 2 * p]) : 1.0f;
      sn[e] = in ? to_f32(ct[row * a.dim + 2 * p + 1]) : 0.0f;
    } else {
      cs[e] = in ? to_f32(ct[row * half + p]) : 1.0f;
      sn[e] = in ? to_f32(st[row * half + p]) : 0.0f;
    }
  }
  return stay;
}

// VEC elements of x per slot (a slot and its partner with HALF); XVEC: slots
// of x and out start on their own size.
template <typename XT, typename TT, typename OT, int VEC, bool HALF, bool PACKED, bool XVEC,
          bool TVEC, int HPT>
__device__ __forceinline__ void rope_positions(const RopePosArgs& a) {
  constexpr int NP = HALF ? VEC : VEC / 2;           // pairs per slot
  constexpr int PARTS = HALF ? 2 : 1;
  const int spr = (a.dim / 2) / NP;                  // slots (of pairs) per head
  const int j = threadIdx.x % spr;
  const int rest = threadIdx.x / spr;
  const int hl = rest % a.head_lanes, tl = rest / a.head_lanes;
  const long long token = (long long)blockIdx.x * a.tokens_per_cta + tl;
  if (tl >= a.tokens_per_cta || token >= a.tokens) return;
  const int p0 = j * NP;
  const int e0 = HALF ? p0 : 2 * p0;                 // first element of the slot
  const XT* x = static_cast<const XT*>(a.x) + token * a.x_token + e0;
  OT* out = static_cast<OT*>(a.out) + token * a.heads * (long long)a.dim + e0;
  float cs[NP], sn[NP];
  bool have = false;
  for (int h0 = hl; h0 < a.heads; h0 += a.head_lanes * HPT) {
    Slot<XT, VEC> s[HPT][PARTS];
#pragma unroll
    for (int u = 0; u < HPT; ++u) {
      const int h = h0 + u * a.head_lanes;
      if (h >= a.heads) break;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        const XT* src = x + h * a.x_head + p * (a.dim / 2);
        if constexpr (XVEC) {
          s[u][p] = load_slot<kLoadInPlace, XT, VEC>(src);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) s[u][p].v[e] = src[e];     // (out may be x: no .nc)
        }
      }
    }
    if (!have) {
      const uint32_t stay = rope_table<TT, NP, PACKED, TVEC>(a, token, p0, cs, sn);
      have = true;
      if (stay != 0u) {
        // padding: a turn by 0 would make NaN of an infinity's partner, and 0 of -0
#pragma unroll 1
        for (int h = hl; h < a.heads; h += a.head_lanes) {
          const XT* src = x + h * a.x_head;
          OT* dst = out + (long long)h * a.dim;
          if constexpr (XVEC) if (stay == (1u << NP) - 1u) {     // (a whole slot: all axes, mostly)
#pragma unroll 1
            for (int p = 0; p < PARTS; ++p) {
              const Slot<XT, VEC> slot = load_slot<kLoadInPlace, XT, VEC>(src + p * (a.dim / 2));
              float f[VEC];
#pragma unroll
              for (int e = 0; e < VEC; ++e) f[e] = to_f32(slot.v[e]);
              Slot<OT, VEC> so;
              pack_slot<OT, VEC>(so, f);
              store_slot<kStoreDefault, OT, VEC>(dst + p * (a.dim / 2), so);
            }
            continue;
          }
#pragma unroll
          for (int e = 0; e < NP; ++e) {
            const int i0 = HALF ? e : 2 * e, i1 = HALF ? e + a.dim / 2 : 2 * e + 1;
            const float v0 = to_f32(src[i0]), v1 = to_f32(src[i1]);
            const bool left = stay >> e & 1u;
            dst[i0] = from_f32<OT>(left ? v0 : v0 * cs[e] - v1 * sn[e]);
            dst[i1] = from_f32<OT>(left ? v1 : v0 * sn[e] + v1 * cs[e]);
          }
        }
        return;
      }
    }
#pragma unroll
    for (int u = 0; u < HPT; ++u) {
      const int h = h0 + u * a.head_lanes;
      if (h >= a.heads) break;
      float o[PARTS][VEC];
#pragma unroll
      for (int e = 0; e < NP; ++e) {
        const float v0 = to_f32(HALF ? s[u][0].v[e] : s[u][0].v[2 * e]);
        const float v1 = to_f32(HALF ? s[u][PARTS - 1].v[e] : s[u][0].v[2 * e + 1]);
        const float r0 = v0 * cs[e] - v1 * sn[e], r1 = v0 * sn[e] + v1 * cs[e];
        if constexpr (HALF) { o[0][e] = r0; o[PARTS - 1][e] = r1; }
        else { o[0][2 * e] = r0; o[0][2 * e + 1] = r1; }
      }
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
        OT* dst = out + (long long)h * a.dim + p * (a.dim / 2);
        if constexpr (XVEC) {
          Slot<OT, VEC> so;
          pack_slot<OT, VEC>(so, o[p]);
          store_slot<kStoreDefault, OT, VEC>(dst, so);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) dst[e] = from_f32<OT>(o[p][e]);
        }
      }
    }
  }
}

}  // namespace molten
