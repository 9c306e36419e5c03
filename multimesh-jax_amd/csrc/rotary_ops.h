// Rotary positions: the work of one workgroup, on a sharded array or on the way into the pages of a cache.
//
// Pair i of a row at position p is turned by the angle 2 pi t, t = p * f_i:
//   y_a = x_a c - x_b s,  y_b = x_b c + x_a s,  c = m cos 2 pi t,  s = m sin 2 pi t
// with (a, b) = (i, i + R/2), or (2i, 2i + 1) interleaved; what stands behind the first R elements passes through.  The
// gradient of the input is the same with s of the other sign, as the matrix is m times a rotation.
//
// Angles.  f_i is held as a fraction of a turn in 64 bits of fixed point, so t modulo 1 is the low half of an integer
// product, of which the upper 32 bits are used: low by under 2^-32 of a turn at any position, and up to 2^-34 off at position
// 2^31 for the rounding of f_i, where a 32-bit float product would be off by many turns.  They are cut into a quarter turn
// and a rest within +-pi/4, and sine and cosine of the rest are their Taylor sums to the 9th and 10th power: cut off under
// 2^-28, rounding 2^-24.
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
constexpr int kRotaryHeads = 4;    // heads a lane takes with one set of angles
constexpr int kRotaryShapes = 3;   // shapes of one call (queries, keys, values)

// n / d for n < 256 and 1 <= d <= 256: exact, as n * (mul * d - 2^16) < n * d < 2^16.
MMR_HD uint32_t small_div(uint32_t n, uint32_t mul) { return (n * mul) >> 16; }
inline uint32_t make_small_div(uint32_t d) { return (65536u + d - 1) / d; }

// Rows of `dim` elements over outer x seq tokens and heads, and how they are dealt to workgroups: the extents of a tile,
// the same on every device.  Strides in bytes.
struct RotaryShape {
  int64_t src_outer, src_seq, src_head;
  int64_t dst_outer, dst_seq, dst_head;  // paged: dst_outer is the page, dst_seq the token of a page
  int64_t pos_outer, pos_seq;            // in elements
  uint32_t tokens, seq, heads;           // tokens = outer * seq
  uint32_t rot_units, units;             // units of a row: rotated ones first
  uint32_t rest_at, rest_bytes;          // the part that passes through
  uint32_t head_groups;                  // workgroups along the heads
  uint32_t blocks;                       // workgroups of a buffer
  uint32_t mul_lanes, mul_head_lanes;    // small_div by the two
  uint16_t lanes;                        // lanes of a row: min(units, kRotaryThreads)
  uint16_t head_lanes;                   // rows of a workgroup along the heads ...
  uint16_t token_lanes;                  // ... and along the tokens
  uint16_t head_steps;                   // heads a lane takes, head_lanes apart
  uint32_t rest_two;                     // a unit of the rest is two vectors, like those of the rotated part
  uint32_t paged;                        // 1: into pages; 2: by the positions of a paged write, beside the source
  FastDiv div_seq, div_head_groups;
};

// One buffer of that shape, and how much of the tile is not padding.
struct RotaryBuffer {
  const char* src;
  char* dst;
  const int32_t* positions;  // null: base + index along seq
  int64_t base;
  uint32_t outer, seq, heads;
  uint32_t shape;
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

struct RotaryAngles {
  const uint64_t* frequency;  // turns per position, 0.64 fixed point
  float magnitude;
  float sine;                 // magnitude, negative for the gradient
  uint32_t half;              // R / 2
};

// The argument block of a launch of up to N buffers of up to S shapes.  Its size is much of what a launch of few rows
// costs: with 3 KB (16 buffers, each with all a shape holds) a layer of a decode step took 6.0 us, and 28 us waited for
// alone; with 0.7 KB 5.7 and 19.  So there are three: one shape on up to 8 devices (0.6 KB), queries, keys and values on
// one device (0.7 KB), and everything else (1.6 KB).
template <int S, int N>
struct RotaryArgs {
  static constexpr int kShapes = S, kBuffers = N;
  RotaryAngles angles;
  RotaryPages pages;
  RotaryShape shapes[S];
  RotaryBuffer buffers[N];
};
typedef RotaryArgs<1, 8> RotaryOneShape;
typedef RotaryArgs<kRotaryShapes, 4> RotaryFewBuffers;
typedef RotaryArgs<kRotaryShapes, 24> RotaryManyBuffers;

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

// The vector of VEC elements a lane turns, as 32-bit words.  Of 16 bytes it is aligned, narrower ones stand anywhere.
template <class T, int VEC>
struct RotaryVec {
  static constexpr int kBytes = VEC * T::kBytes;
  static constexpr int kWords = (kBytes + 3) / 4;
  uint32_t w[kWords] = {};

  template <class M>
  MMR_HD void load(typename M::cptr p) {
    if constexpr (kBytes == 16) {
      const V16 v = M::load16(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (kBytes == 8) {
      const uint64_t v = M::template loadu<uint64_t>(p);
      w[0] = static_cast<uint32_t>(v), w[1] = static_cast<uint32_t>(v >> 32);
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
    else if constexpr (kBytes == 8) M::template storeu<uint64_t>(p, w[0] | static_cast<uint64_t>(w[1]) << 32);
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

// Position and place of token t of a paged write: false if it has none (padding, or a bad entry: *bad).
template <class X>
MMR_HD bool rotary_place(X& x, const RotaryPages& pg, int32_t wave_token, int32_t t, int64_t* position, int32_t* page,
                         int32_t* in_page, uint32_t* bad) {
  // one token a sequence, without padding: entry t (a guess that a step of decoding always gets right saves it one load
  // of the chain, and costs others nothing, as its loads wait for none)
  int32_t entry = t < pg.n ? t : pg.n - 1;
  if (!x.all(pg.begins[entry] <= t && t < pg.begins[entry + 1]))
    entry = x.ended(pg.begins + 1, pg.n, wave_token);  // entries that end at or before the wave's first token
  if (entry < pg.n && pg.begins[entry + 1] <= t) {     // a later token in a later entry
    int32_t lo = entry + 1, hi = pg.n;
    while (lo < hi) {
      const int32_t mid = (lo + hi) >> 1;
      if (pg.begins[mid + 1] <= t) lo = mid + 1;
      else hi = mid;
    }
    entry = lo;
  }
  if (entry >= pg.n) return false;  // behind the last sequence
  const int32_t begin = pg.begins[entry], end = pg.begins[entry + 1], slot = pg.slots[entry];
  if (t < begin) return false;  // before the first one
  if (slot < 0 || slot >= pg.S) {
    *bad = slot == MMR_PAGES_NONE ? 0 : MMR_PAGES_BAD_SEQUENCE;
    return false;
  }
  const int64_t p = static_cast<int64_t>(pg.lengths[slot]) - end + t;
  if (p < 0 || p >= pg.capacity) {
    *bad = MMR_PAGES_TOO_LONG;
    return false;
  }
  const int32_t at = static_cast<int32_t>(fdiv(static_cast<uint32_t>(p), pg.div_T));
  *position = p;
  *in_page = static_cast<int32_t>(p) - at * pg.T;
  *page = pg.table[static_cast<int64_t>(slot) * pg.B + at];
  if (*page < 0 || *page >= pg.P) *bad = MMR_PAGES_BAD_PAGE;
  return *bad == 0;
}

// Lane (row, unit) of workgroup `block` of a buffer.  A unit is what a lane turns: the two vectors that hold VEC pairs, or,
// interleaved, one vector of VEC / 2 pairs; in the rest of the row it is two vectors as well, where they are whole ones of
// 16 bytes (half of bf16 rows of 128 turned: 37.0 -> 34.4 us for 12,000 tokens of 32 heads), and otherwise 16 bytes, the last ones slid back to end with the
// row (they repeat their neighbour's bytes, with the same values), or one element if the rest is shorter.  The rows are
// loaded before the position is looked up: the look-up is a chain of four loads.
template <class M, class T, int VEC, bool INTERLEAVED, class X>
MMR_HD void rotary_block(X& x, const RotaryAngles& a, const RotaryPages& pages, const RotaryShape& j, const RotaryBuffer& b) {
  constexpr int kVecBytes = VEC * T::kBytes;
  static_assert(!INTERLEAVED || VEC > 1, "an interleaved unit holds whole pairs");
  constexpr bool kTwo = T::kBytes > 1 && !INTERLEAVED;  // a unit of the rotated part is two vectors
  constexpr int kPairs = INTERLEAVED ? VEC / 2 : VEC;   // and so many pairs
  constexpr bool kWide = kVecBytes == 16;               // every row and the rest of it are whole aligned vectors
  const uint32_t group = fdiv(x.block, j.div_head_groups), hg = x.block - group * j.head_groups;
  const uint32_t row = small_div(static_cast<uint32_t>(x.tid), j.mul_lanes), lane = static_cast<uint32_t>(x.tid) - row * j.lanes;
  const uint32_t tsub = small_div(row, j.mul_head_lanes), hsub = row - tsub * j.head_lanes;
  const uint32_t token = group * j.token_lanes + tsub;
  const bool inside = tsub < j.token_lanes && token < j.tokens;
  const uint32_t outer = fdiv(inside ? token : 0u, j.div_seq), seq = (inside ? token : 0u) - outer * j.seq;
  const bool on = inside && outer < b.outer && seq < b.seq;
  const char* const src = b.src + (static_cast<int64_t>(outer) * j.src_outer + static_cast<int64_t>(seq) * j.src_seq);
  const uint32_t h0 = hg * j.head_lanes * j.head_steps + hsub;

  // byte offsets in a row of the two vectors of a unit (of the one, for units of the rest)
  auto offsets = [&](uint32_t unit, int64_t* off_a, int64_t* off_b) {
    if (unit < j.rot_units) {
      *off_a = static_cast<int64_t>(unit) * kVecBytes;
      *off_b = *off_a + static_cast<int64_t>(a.half) * T::kBytes;
    } else {
      const uint32_t at = unit - j.rot_units;
      if (kTwo && kWide && j.rest_two) {
        *off_a = static_cast<int64_t>(j.rest_at) + at * 16;
        *off_b = *off_a + j.rest_bytes / 2;
        return;
      }
      uint32_t in_rest = at * T::kBytes;
      if (j.rest_bytes >= 16) in_rest = at * 16 + 16 <= j.rest_bytes ? at * 16 : j.rest_bytes - 16;
      *off_a = *off_b = static_cast<int64_t>(j.rest_at) + in_rest;
    }
  };
  RotaryVec<T, VEC> va[kRotaryHeads], vb[kRotaryHeads];
  V16 rest[kRotaryHeads];  // where the vectors are narrower
  auto load = [&](uint32_t unit) {
    int64_t off_a, off_b;
    offsets(unit, &off_a, &off_b);
#pragma unroll
    for (uint32_t k = 0; k < kRotaryHeads; ++k) {
      const uint32_t h = h0 + k * j.head_lanes;
      if (k < j.head_steps && h < b.heads) {
        const typename M::cptr from = M::cplace(src + (h * j.src_head + off_a));
        if (kWide || unit < j.rot_units) va[k].template load<M>(from);
        else if (j.rest_bytes >= 16) rest[k] = M::load16u(from);
        else if (T::kBytes == 4) rest[k].x = M::template loadu<uint32_t>(from);
        else if (T::kBytes == 2) rest[k].x = M::template loadu<uint16_t>(from);
        else rest[k].x = M::template loadu<uint8_t>(from);
        if (kTwo && (unit < j.rot_units || (kWide && j.rest_two))) vb[k].template load<M>(M::cplace(src + (h * j.src_head + off_b)));
      }
    }
  };
  uint64_t f[kPairs];
  auto load_frequencies = [&](uint32_t unit) {
    if (T::kBytes > 1 && unit < j.rot_units) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) f[i] = a.frequency[unit * kPairs + i];
    }
  };
  if (on) {
    load(lane);
    load_frequencies(lane);
  }

  int64_t position = 0;
  char* dst = b.dst;
  if (j.paged) {
    // the token of the wave's first lane, for all lanes to look up together
    const uint32_t first = small_div(small_div(static_cast<uint32_t>(x.tid) & ~63u, j.mul_lanes), j.mul_head_lanes);
    const uint32_t ask = group * j.token_lanes + first;
    const int32_t wave_token = static_cast<int32_t>(ask < j.tokens ? ask : j.tokens - 1);
    int32_t page = 0, in_page = 0;
    uint32_t bad = 0;
    // lanes without a token ask for their wave's first one and go no further
    const bool there = rotary_place(x, pages, wave_token, on ? static_cast<int32_t>(token) : wave_token, &position, &page, &in_page, &bad);
    if (!on) return;
    if (!there) {
      if (bad && lane == 0 && hsub == 0) x.atomic_or(pages.status, static_cast<int32_t>(bad));
      return;
    }
    if (j.paged == 1) dst += static_cast<int64_t>(page) * j.dst_outer + static_cast<int64_t>(in_page) * j.dst_seq;
    else dst += static_cast<int64_t>(seq) * j.dst_seq;  // queries: turned by the token's position, written beside it
  } else {
    if (!on) return;
    position = b.positions ? b.positions[static_cast<int64_t>(outer) * j.pos_outer + static_cast<int64_t>(seq) * j.pos_seq]
                           : b.base + seq;
    dst += static_cast<int64_t>(outer) * j.dst_outer + static_cast<int64_t>(seq) * j.dst_seq;
  }

  for (uint32_t unit = lane;;) {
    int64_t off_a, off_b;
    offsets(unit, &off_a, &off_b);
    if (T::kBytes > 1 && unit < j.rot_units) {
      float s[kPairs], c[kPairs];
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        turn_sincos(turns_at(position, f[i]), &s[i], &c[i]);
        s[i] *= a.sine;
        c[i] *= a.magnitude;
      }
#pragma unroll
      for (uint32_t k = 0; k < kRotaryHeads; ++k) {
        if (k >= j.head_steps) break;  // uniform over the launch
        if constexpr (VEC == 1) {
          const float xa = va[k].get(0), xb = vb[k].get(0);
          va[k].put1(xa * c[0] - xb * s[0]);
          vb[k].put1(xb * c[0] + xa * s[0]);
        } else if constexpr (INTERLEAVED) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            const float xa = va[k].get(2 * i), xb = va[k].get(2 * i + 1);
            va[k].put2(2 * i, xa * c[i] - xb * s[i], xb * c[i] + xa * s[i]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < VEC; e += 2) {
            const float a0 = va[k].get(e), a1 = va[k].get(e + 1), b0 = vb[k].get(e), b1 = vb[k].get(e + 1);
            va[k].put2(e, a0 * c[e] - b0 * s[e], a1 * c[e + 1] - b1 * s[e + 1]);
            vb[k].put2(e, b0 * c[e] + a0 * s[e], b1 * c[e + 1] + a1 * s[e + 1]);
          }
        }
        const uint32_t h = h0 + k * j.head_lanes;
        if (h < b.heads) {
          va[k].template store<M>(M::place(dst + (h * j.dst_head + off_a)));
          if (kTwo) vb[k].template store<M>(M::place(dst + (h * j.dst_head + off_b)));
        }
      }
    } else {
#pragma unroll
      for (uint32_t k = 0; k < kRotaryHeads; ++k) {
        const uint32_t h = h0 + k * j.head_lanes;
        if (k >= j.head_steps || h >= b.heads) continue;
        const typename M::ptr to = M::place(dst + (h * j.dst_head + off_a));
        if (kWide) {
          va[k].template store<M>(to);
          if (kTwo && j.rest_two) vb[k].template store<M>(M::place(dst + (h * j.dst_head + off_b)));
        }
        else if (j.rest_bytes >= 16) M::template storeu<V16>(to, rest[k]);
        else if (T::kBytes == 4) M::template storeu<uint32_t>(to, rest[k].x);
        else if (T::kBytes == 2) M::template storeu<uint16_t>(to, static_cast<uint16_t>(rest[k].x));
        else M::template storeu<uint8_t>(to, static_cast<uint8_t>(rest[k].x));
      }
    }
    unit += j.lanes;
    if (unit >= j.units) break;
    load(unit);
    load_frequencies(unit);
  }
}

// Units of a row of `bytes` bytes with `turned` of them turned, in units of `unit_bytes`; `element`: bytes of one.
inline void rotary_units(RotaryShape* j, uint32_t bytes, uint32_t turned, uint32_t unit_bytes, uint32_t element, bool in_place) {
  j->rot_units = turned / unit_bytes;
  j->rest_at = turned;
  j->rest_bytes = in_place ? 0 : bytes - turned;  // in place, what is not turned stays
  j->rest_two = element > 1 && unit_bytes == 32 && j->rest_bytes > 0 && j->rest_bytes % 32 == 0;
  j->units = j->rot_units + (j->rest_two ? j->rest_bytes / 32 : j->rest_bytes >= 16 ? (j->rest_bytes + 15) / 16 : j->rest_bytes / element);
}

// How the rows of a shape are dealt to workgroups; returns how many that takes.  `spread`: one head a lane, for launches
// that would not fill the chip.
inline uint64_t rotary_shape(RotaryShape* j, bool heads_adjacent, bool spread) {
  const uint32_t threads = kRotaryThreads;
  const uint32_t lanes = j->units < threads ? j->units : threads;
  const uint32_t rows = threads / lanes;
  const uint32_t want = spread ? 1u : static_cast<uint32_t>(kRotaryHeads);
  uint32_t head_lanes = heads_adjacent || spread ? (j->heads + want - 1) / want : 1;
  if (head_lanes > rows) head_lanes = rows;
  uint32_t token_lanes = rows / head_lanes;
  if (spread && j->tokens < 1024) token_lanes = 1;
  const uint32_t steps = (j->heads + head_lanes - 1) / head_lanes;
  const uint32_t groups = (steps + want - 1) / want;
  const uint32_t head_steps = (steps + groups - 1) / groups;  // 5 heads go as 3 and 2, not as 4 and 1
  const uint32_t per = head_lanes * head_steps;
  j->head_groups = (j->heads + per - 1) / per;
  const uint64_t blocks = (static_cast<uint64_t>(j->tokens) + token_lanes - 1) / token_lanes * j->head_groups;
  j->blocks = static_cast<uint32_t>(blocks);
  j->lanes = static_cast<uint16_t>(lanes), j->head_lanes = static_cast<uint16_t>(head_lanes);
  j->token_lanes = static_cast<uint16_t>(token_lanes), j->head_steps = static_cast<uint16_t>(head_steps);
  j->mul_lanes = make_small_div(lanes), j->mul_head_lanes = make_small_div(head_lanes);
  j->div_seq = make_fastdiv(j->seq);
  j->div_head_groups = make_fastdiv(j->head_groups);
  return blocks;
}

}  // namespace mmr

#endif  // MMR_CSRC_ROTARY_OPS_H_
