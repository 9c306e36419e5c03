// Rotary positions: the work of one workgroup, on a sharded array or on the way into the pages of a cache.
//
// Pair i of a row at position p is turned by the angle 2 pi t, t = p * f_i:
//   y_a = x_a c - x_b s,  y_b = x_b c + x_a s,  c = m cos 2 pi t,  s = m sin 2 pi t
// with (a, b) = (i, i + R/2), or (2i, 2i + 1) interleaved; what stands behind the first R elements passes through.  The
// gradient of the input is the same with s of the other sign, as the matrix is m times a rotation.
//
// Angles.  f_i is held as a fraction of a turn in 64 bits of fixed point, so t modulo 1 is the low half of an integer
// product and nothing is lost at far positions (2^-34 of a turn at position 2^31, where a 32-bit float product would be
// off by many turns).  Its upper 32 bits are cut into a quarter turn and a rest within +-pi/4, and sine and cosine of
// the rest are their Taylor sums to the 9th and 10th power: cut off under 2^-28, rounding 2^-24.
//
// Bound: HBM; a row is read and written once.  The angles of a position are worked out once per lane and used for
// several heads, so that their ~35 instructions a pair stay below the time of the memory traffic.
#ifndef MMR_CSRC_ROTARY_OPS_H_
#define MMR_CSRC_ROTARY_OPS_H_

#include <cstdint>

#include "group_ops.h"
#include "page_ops.h"

namespace mmr {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryHeads = 4;   // heads a lane takes with one set of angles
constexpr int kRotaryMaxJobs = 16;

// One buffer: rows of `dim` elements over outer x seq tokens and heads.  Strides in bytes.
struct RotaryJob {
  const char* src;
  char* dst;
  int64_t src_outer, src_seq, src_head;
  int64_t dst_outer, dst_seq, dst_head;  // paged: dst_outer is the page, dst_seq the token of a page
  const int32_t* positions;              // null: base + index along seq
  int64_t pos_outer, pos_seq;
  int64_t base;
  uint32_t tokens, seq, heads;  // tokens = outer * seq
  uint32_t rot_units, units;    // units of a row: rotated ones first
  uint32_t lanes;               // lanes of a row: min(units, kRotaryThreads)
  uint32_t head_lanes;          // rows of a workgroup along the heads ...
  uint32_t token_lanes;         // ... and along the tokens
  uint32_t head_steps;          // heads a lane takes, head_lanes apart
  uint32_t head_groups;         // workgroups along the heads
  uint32_t blocks;              // workgroups of this job
  uint32_t paged;
  FastDiv div_seq, div_lanes, div_head_lanes, div_head_groups;
};

// Where new tokens of a paged write go.
struct RotaryPages {
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* slots;
  const int32_t* begins;
  int32_t* status;
  int32_t n, S, B, P, T;
  int32_t capacity;
  FastDiv div_T;
};

struct RotaryArgs {
  const uint64_t* frequency;  // turns per position, 0.64 fixed point
  float magnitude;
  float sine;                 // magnitude, negative for the gradient
  uint32_t half;              // R / 2
  RotaryPages pages;
  RotaryJob jobs[kRotaryMaxJobs];
};

// sin and cos of `turns` / 2^32 of a turn
MMR_HD void turn_sincos(uint32_t turns, float* s, float* c) {
  const uint32_t quarter = (turns + 0x20000000u) >> 30;
  const int32_t rest = static_cast<int32_t>(turns - (quarter << 30));
  const float y = static_cast<float>(rest) * 1.46291807926715968e-9f;  // 2 pi / 2^32
  const float z = y * y;
  const float sp = y + y * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
  const float cp = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
  const float sv = (quarter & 1) ? cp : sp, cv = (quarter & 1) ? sp : cp;
  *s = (quarter & 2) ? -sv : sv;
  *c = ((quarter + 1) & 2) ? -cv : cv;
}

MMR_HD uint32_t turns_at(int64_t position, uint64_t frequency) {
  return static_cast<uint32_t>((static_cast<uint64_t>(position) * frequency) >> 32);
}

// Element types.  VEC elements: one 16-byte vector, or a single element.
struct RotaryRaw {  // bytes that only move
  static constexpr int kBytes = 1;
  static MMR_HD float get(uint32_t) { return 0.0f; }
  static MMR_HD uint32_t put(float) { return 0; }
};
struct RotaryF32 {
  static constexpr int kBytes = 4;
  static MMR_HD float get(uint32_t v) { return __builtin_bit_cast(float, v); }
  static MMR_HD uint32_t put(float v) { return __builtin_bit_cast(uint32_t, v); }
};
struct RotaryBF16 {
  static constexpr int kBytes = 2;
  static MMR_HD float get(uint32_t v) { return __builtin_bit_cast(float, v << 16); }
  static MMR_HD uint32_t put(float v) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)); }  // to nearest even
};
struct RotaryF16 {
  static constexpr int kBytes = 2;
  static MMR_HD float get(uint32_t v) { return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(v))); }
  static MMR_HD uint32_t put(float v) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v)); }
};

// The 16-byte (or one-element) vector a lane holds, as 32-bit words.
template <class T, int VEC>
struct RotaryVec {
  static constexpr int kBytes = VEC * T::kBytes;
  static constexpr int kWords = (kBytes + 3) / 4;
  uint32_t w[kWords];

  template <class M>
  MMR_HD void load(typename M::cptr p) {
    if constexpr (kBytes == 16) {
      const V16 v = M::load16(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (kBytes == 4) {
      w[0] = M::template loadu<uint32_t>(p);
    } else if constexpr (kBytes == 2) {
      w[0] = M::template loadu<uint16_t>(p);
    } else {
      w[0] = M::template loadu<uint8_t>(p);
    }
  }
  template <class M>
  MMR_HD void store(typename M::ptr p) const {
    if constexpr (kBytes == 16) M::store16(p, V16{w[0], w[1], w[2], w[3]});
    else if constexpr (kBytes == 4) M::template storeu<uint32_t>(p, w[0]);
    else if constexpr (kBytes == 2) M::template storeu<uint16_t>(p, static_cast<uint16_t>(w[0]));
    else M::template storeu<uint8_t>(p, static_cast<uint8_t>(w[0]));
  }
  MMR_HD float get(int i) const {
    if constexpr (T::kBytes == 4) return T::get(w[i]);
    else if constexpr (T::kBytes == 2) return T::get((w[i / 2] >> (i % 2 * 16)) & 0xffffu);
    else return 0.0f;
  }
  MMR_HD void put2(int i, float a, float b) {  // elements i (even) and i + 1
    if constexpr (T::kBytes == 4) w[i] = T::put(a), w[i + 1] = T::put(b);
    else if constexpr (T::kBytes == 2) w[i / 2] = T::put(a) | (T::put(b) << 16);
  }
  MMR_HD void put1(float a) { w[0] = T::put(a); }  // VEC == 1
};

// Lane (row, unit) of workgroup `block` of a job.  A unit is two vectors (VEC pairs) of the rotated part, or one vector
// of the rest.
template <class M, class T, int VEC, bool INTERLEAVED, class X>
MMR_HD void rotary_block(X& x, const RotaryArgs& a, const RotaryJob& j) {
  constexpr int kVecBytes = VEC * T::kBytes;
  const uint32_t group = fdiv(x.block, j.div_head_groups), hg = x.block - group * j.head_groups;
  const uint32_t row = fdiv(static_cast<uint32_t>(x.tid), j.div_lanes), lane = static_cast<uint32_t>(x.tid) - row * j.lanes;
  const uint32_t tsub = fdiv(row, j.div_head_lanes), hsub = row - tsub * j.head_lanes;
  const uint32_t t0 = group * j.token_lanes, token = t0 + tsub;
  bool on = tsub < j.token_lanes && token < j.tokens;

  int64_t position = 0;
  const char* src = j.src;
  char* dst = j.dst;
  if (j.paged) {
    // entry of the workgroup's first token: how many entries end at or before it (all threads, two barriers)
    const RotaryPages& pg = a.pages;
    int32_t ended = 0, entry = 0;
    for (int32_t i = x.tid; i < pg.n; i += kRotaryThreads) ended += pg.begins[i + 1] <= static_cast<int32_t>(t0);
    x.scan(ended, &entry);
    if (!on) return;
    const int32_t t = static_cast<int32_t>(token);
    if (entry < pg.n && pg.begins[entry + 1] <= t) {  // a later token of the workgroup in a later entry
      int32_t lo = entry + 1, hi = pg.n;
      while (lo < hi) {
        const int32_t mid = (lo + hi) >> 1;
        if (pg.begins[mid + 1] <= t) lo = mid + 1;
        else hi = mid;
      }
      entry = lo;
    }
    if (entry >= pg.n) return;  // behind the last sequence
    const int32_t begin = pg.begins[entry], end = pg.begins[entry + 1], slot = pg.slots[entry];
    if (t < begin) return;  // before the first one
    uint32_t bad = 0;
    int32_t page = 0, in_page = 0;
    if (slot < 0 || slot >= pg.S) {
      bad = MMR_PAGES_BAD_SEQUENCE;
    } else {
      const int64_t p = static_cast<int64_t>(pg.lengths[slot]) - (static_cast<int64_t>(end) - begin) + (static_cast<int64_t>(t) - begin);
      if (p < 0 || p >= pg.capacity) {
        bad = MMR_PAGES_TOO_LONG;
      } else {
        position = p;
        const int32_t at = static_cast<int32_t>(fdiv(static_cast<uint32_t>(p), pg.div_T));
        in_page = static_cast<int32_t>(p) - at * pg.T;
        page = pg.table[static_cast<int64_t>(slot) * pg.B + at];
        if (page < 0 || page >= pg.P) bad = MMR_PAGES_BAD_PAGE;
      }
    }
    if (bad) {
      if (lane == 0 && hsub == 0) x.atomic_or(pg.status, static_cast<int32_t>(bad));
      return;
    }
    src += static_cast<int64_t>(token) * j.src_seq;
    if (j.paged == 1) dst += static_cast<int64_t>(page) * j.dst_outer + static_cast<int64_t>(in_page) * j.dst_seq;
    else dst += static_cast<int64_t>(token) * j.dst_seq;  // queries: turned by the token's position, written beside it
  } else {
    if (!on) return;
    const uint32_t outer = fdiv(token, j.div_seq), s = token - outer * j.seq;
    position = j.positions ? j.positions[static_cast<int64_t>(outer) * j.pos_outer + static_cast<int64_t>(s) * j.pos_seq]
                           : j.base + s;
    src += static_cast<int64_t>(outer) * j.src_outer + static_cast<int64_t>(s) * j.src_seq;
    dst += static_cast<int64_t>(outer) * j.dst_outer + static_cast<int64_t>(s) * j.dst_seq;
  }

  const uint32_t h0 = hg * j.head_lanes * j.head_steps + hsub;
  for (uint32_t unit = lane; unit < j.units; unit += j.lanes) {
    if (unit >= j.rot_units) {
      const int64_t off = (2 * static_cast<int64_t>(j.rot_units) + (unit - j.rot_units)) * kVecBytes;
      for (uint32_t i = 0; i < j.head_steps; i += kRotaryHeads) {
        RotaryVec<T, VEC> v[kRotaryHeads];
#pragma unroll
        for (uint32_t k = 0; k < kRotaryHeads; ++k) {
          const uint32_t h = h0 + (i + k) * j.head_lanes;
          if (i + k < j.head_steps && h < j.heads) v[k].template load<M>(M::cplace(src + (h * j.src_head + off)));
        }
#pragma unroll
        for (uint32_t k = 0; k < kRotaryHeads; ++k) {
          const uint32_t h = h0 + (i + k) * j.head_lanes;
          if (i + k < j.head_steps && h < j.heads) v[k].template store<M>(M::place(dst + (h * j.dst_head + off)));
        }
      }
      continue;
    }
    if constexpr (T::kBytes > 1) {
      // byte offsets of the unit's two vectors and the pairs they hold
      int64_t off_a, off_b;
      if (INTERLEAVED && VEC == 1) off_a = static_cast<int64_t>(2) * unit * kVecBytes, off_b = off_a + kVecBytes;
      else off_a = static_cast<int64_t>(unit) * kVecBytes, off_b = off_a + static_cast<int64_t>(a.half) * T::kBytes;
      float s[VEC], c[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        uint32_t pair;
        if (!INTERLEAVED || VEC == 1) pair = unit * VEC + i;
        else pair = i < VEC / 2 ? unit * (VEC / 2) + i : (a.half + unit * VEC) / 2 + (i - VEC / 2);
        turn_sincos(turns_at(position, a.frequency[pair]), &s[i], &c[i]);
        s[i] *= a.sine;
        c[i] *= a.magnitude;
      }
      for (uint32_t i = 0; i < j.head_steps; i += kRotaryHeads) {
        RotaryVec<T, VEC> va[kRotaryHeads], vb[kRotaryHeads];
#pragma unroll
        for (uint32_t k = 0; k < kRotaryHeads; ++k) {
          const uint32_t h = h0 + (i + k) * j.head_lanes;
          if (i + k < j.head_steps && h < j.heads) {
            va[k].template load<M>(M::cplace(src + (h * j.src_head + off_a)));
            vb[k].template load<M>(M::cplace(src + (h * j.src_head + off_b)));
          }
        }
#pragma unroll
        for (uint32_t k = 0; k < kRotaryHeads; ++k) {
          const uint32_t h = h0 + (i + k) * j.head_lanes;
          if (i + k >= j.head_steps || h >= j.heads) continue;
          if constexpr (VEC == 1) {
            const float xa = va[k].get(0), xb = vb[k].get(0);
            va[k].put1(xa * c[0] - xb * s[0]);
            vb[k].put1(xb * c[0] + xa * s[0]);
          } else if constexpr (INTERLEAVED) {
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
              const float a0 = va[k].get(e), b0 = va[k].get(e + 1), a1 = vb[k].get(e), b1 = vb[k].get(e + 1);
              const float c0 = c[e / 2], s0 = s[e / 2], c1 = c[VEC / 2 + e / 2], s1 = s[VEC / 2 + e / 2];
              va[k].put2(e, a0 * c0 - b0 * s0, b0 * c0 + a0 * s0);
              vb[k].put2(e, a1 * c1 - b1 * s1, b1 * c1 + a1 * s1);
            }
          } else {
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
              const float a0 = va[k].get(e), a1 = va[k].get(e + 1), b0 = vb[k].get(e), b1 = vb[k].get(e + 1);
              va[k].put2(e, a0 * c[e] - b0 * s[e], a1 * c[e + 1] - b1 * s[e + 1]);
              vb[k].put2(e, b0 * c[e] + a0 * s[e], b1 * c[e + 1] + a1 * s[e + 1]);
            }
          }
          va[k].template store<M>(M::place(dst + (h * j.dst_head + off_a)));
          vb[k].template store<M>(M::place(dst + (h * j.dst_head + off_b)));
        }
      }
    }
  }
}

// How a job's rows are dealt to workgroups; returns how many that takes.  `spread`: one head a lane, for launches that
// would not fill the chip.
inline uint64_t rotary_shape(RotaryJob* j, uint32_t rot_units, uint32_t rest_units, bool heads_adjacent, bool spread) {
  const uint32_t threads = kRotaryThreads;
  j->rot_units = rot_units;
  j->units = rot_units + rest_units;
  j->lanes = j->units < threads ? j->units : threads;
  const uint32_t rows = threads / j->lanes;
  const uint32_t want = spread ? 1u : static_cast<uint32_t>(kRotaryHeads);
  j->head_lanes = heads_adjacent || spread ? (j->heads + want - 1) / want : 1;
  if (j->head_lanes > rows) j->head_lanes = rows;
  j->token_lanes = rows / j->head_lanes;
  if (spread && j->token_lanes > 1 && j->tokens < 1024) j->token_lanes = 1;
  j->head_steps = (j->heads + j->head_lanes - 1) / j->head_lanes;
  if (j->head_steps > want) j->head_steps = want;
  const uint32_t per = j->head_lanes * j->head_steps;
  j->head_groups = (j->heads + per - 1) / per;
  const uint64_t blocks = (static_cast<uint64_t>(j->tokens) + j->token_lanes - 1) / j->token_lanes * j->head_groups;
  j->blocks = static_cast<uint32_t>(blocks);
  j->div_seq = make_fastdiv(j->seq);
  j->div_lanes = make_fastdiv(j->lanes);
  j->div_head_lanes = make_fastdiv(j->head_lanes);
  j->div_head_groups = make_fastdiv(j->head_groups);
  return blocks;
}

}  // namespace mmr

#endif  // MMR_CSRC_ROTARY_OPS_H_
