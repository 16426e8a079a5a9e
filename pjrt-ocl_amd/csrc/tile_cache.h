// TOP_CACHE_APPEND, TOP_CACHE_READ (extensions): rows of keys and values into the
// pages of a cache, in place, and back out of them.
//
// A step's rows are described on the device: sequence s's new rows are cu[s] ..
// cu[s + 1] - 1 and its length with them lens[s], so row r is position p = lens[s] -
// (cu[s + 1] - r); it lies in page table[s][p / P] at slot p % P.  Pages are [N,
// heads, P, hd].  A row that belongs to no sequence, whose sequence's length is less
// than its new rows or more than the table holds, or whose table entry is no page of
// the pool has no place: append skips it, read gives zeros.  No entry of cu, lens or
// table can lead an access out of the pages.
//
// i8 pages: q = rint(x / scale), scale = max|x| * (1/127) of the row, one f32 per
// (page, head, slot); read gives q * scale.  A row with an infinity or NaN gets the
// scale NaN (it reads as NaN), a row of zeros the scale 0.  Quotients are correctly
// rounded divisions, so a row's bytes do not depend on how it is computed.
//
// A tile is p7 & 255 rows (64 at most), keys and values of every head.  Each wave looks the
// rows' places up (two dependent reads), and then groups of LPH lanes, 8 channels each, move
// the tile's (row, k or v, head) rows: 16 loads in flight a lane (of f32 eight), kept in LDS while
// the next are on their way and a short loop stores them (one that is unrolled over as many
// rows took as long: every lane runs it once, as fast as its instructions come from memory).
// 4096 rows of 8 heads of 128 from bf16: into bf16 pages 5.8 us a lane (33.5 MB: HBM), into i8
// pages 11 (the conversion's instructions), out of those into f32 13 (42 MB, and 3.5 us until
// the first loads have their rows' places).
#pragma once
#include "tile_rotary.h"
#include "vm_divu32.h"

namespace vm {

struct PagedDesc {
  uint32_t T, Hq, Hkv, hd, P, N, B, MP, cdt;
  uint32_t ars, ahs, aoff, brs, bhs, boff;
  float scale;
  uint32_t window;
  DivU32 dp, dg;       // by P, by Hq / Hkv
};
VM_DEV PagedDesc paged_desc(Args A, const VM_K Task& t) {
  const VM_K int32_t* d = aux_of(A) + t.p[6];
  return PagedDesc{uint32_t(d[PD_T]), uint32_t(d[PD_HQ]), uint32_t(d[PD_HKV]), uint32_t(d[PD_HD]), uint32_t(d[PD_PAGE]),
                   uint32_t(d[PD_PAGES]), uint32_t(d[PD_SEQS]), uint32_t(d[PD_MAXP]), uint32_t(d[PD_CDT]),
                   uint32_t(d[PD_ARS]), uint32_t(d[PD_AHS]), uint32_t(d[PD_AOFF]), uint32_t(d[PD_BRS]),
                   uint32_t(d[PD_BHS]), uint32_t(d[PD_BOFF]), __int_as_float(d[PD_SCALE]), uint32_t(d[PD_WINDOW]),
                   DivU32{uint32_t(d[PD_DIVP]), uint32_t(d[PD_DIVP + 1]), uint32_t(d[PD_DIVP + 2]), uint32_t(d[PD_DIVP + 3])},
                   DivU32{uint32_t(d[PD_DIVG]), uint32_t(d[PD_DIVG + 1]), uint32_t(d[PD_DIVG + 2]), uint32_t(d[PD_DIVG + 3])}};
}

constexpr uint32_t kNoPlace = ~0u;       // (the pages have less than 2^32 rows)

// Places of rows r0 .. r0 + nr - 1 (nr <= 64), lane i's of row r0 + i (past them, of the last): the
// row of the pages [N, heads, P, hd] that head 0's part goes to, or kNoPlace.  A row's sequence is the number of ends cu[1 ..]
// at or before it, counted for 64 sequences at once; their cu and lens arrive together, the
// table entry after them.  Every lane of the wave calls it.
VM_DEV uint32_t row_places(const PagedDesc& D, const VM_G int32_t* cu, const VM_G int32_t* lens,
                           const VM_G int32_t* table, uint32_t r0, uint32_t nr) {
  const uint32_t lane = threadIdx.x & 63, mine = min(lane, nr - 1), r = r0 + mine;
  uint32_t s = 0;
  int32_t c0 = 0, c1 = 0, len = 0;
  for (uint32_t i0 = 0; i0 < D.B; i0 += 64) {
    const uint32_t i = min(i0 + lane, D.B - 1);
    const int32_t a = cu[i], e = cu[i + 1], n = lens[i];
    const bool there = i0 + lane < D.B;
    uint32_t here = 0;                                  // ends of these 64 at or before the lane's row
    for (uint32_t k = 0; k < nr; ++k) {
      const uint32_t c = uint32_t(__builtin_popcountll(__ballot(there && e <= int32_t(r0 + k))));
      here = k == mine ? c : here;
    }
    // the sequence after those, if it is one of these
    const bool hit = s == i0 && here < min(64u, D.B - i0);
    const int32_t a1 = __shfl(a, here & 63, 64), e1 = __shfl(e, here & 63, 64), n1 = __shfl(n, here & 63, 64);
    c0 = hit ? a1 : c0;
    c1 = hit ? e1 : c1;
    len = hit ? n1 : len;
    s += here;
  }
  if (s >= D.B || c0 < 0 || c0 > int32_t(r) || c1 <= int32_t(r) || uint32_t(c1) > D.T) return kNoPlace;
  const uint32_t cap = D.MP * D.P;
  if (len < c1 - c0 || uint32_t(len) > cap) return kNoPlace;
  const uint32_t p = uint32_t(len) - (uint32_t(c1) - r);
  const uint32_t e = D.dp.quo(p);
  const int32_t page = table[uint64_t(s) * D.MP + e];
  if (page < 0 || uint32_t(page) >= D.N) return kNoPlace;
  return uint32_t(page) * D.Hkv * D.P + (p - e * D.P);
}

// Eight signed bytes as f32.
VM_DEV void i8_get(v2u w, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = float(int32_t((i < 4 ? w.x : w.y) << (24 - 8 * (i & 3))) >> 24);
}
// Maximum over the LPH (a power of two) adjacent lanes of a head, of bits that order as
// unsigned numbers, of V heads.
template <int V>
VM_DEV void head_max(uint32_t (&x)[V], uint32_t lph) {
  if (lph > 1)
#pragma unroll
    for (int k = 0; k < V; ++k) x[k] = max(x[k], __float_as_uint(dpp<0xB1>(__uint_as_float(x[k]))));
  if (lph > 2)
#pragma unroll
    for (int k = 0; k < V; ++k) x[k] = max(x[k], __float_as_uint(dpp<0x4E>(__uint_as_float(x[k]))));
  for (uint32_t m = 4; m < lph; m <<= 1)
#pragma unroll
    for (int k = 0; k < V; ++k) x[k] = max(x[k], uint32_t(__shfl_xor(int(x[k]), m, 64)));
}

// Eight elements each of V rows as bytes and, in every lane of the head, the rows' scales.
// The largest |x| is that of the bits without the sign (infinities and NaN are the largest),
// in pairs for 16-bit types.  x / s is x y, y = 1 / s rounded, corrected twice by its
// remainder: with the remainders exact (no underflow for the scales taken here) the second
// correction rounds the quotient correctly (Markstein).  Seven instructions an element with
// the rounding to an integer, by adding 1.5 * 2^23, whose low byte is the integer's; the
// general division takes some 12 more.  (Rounding x y itself and dividing only where that is within 2^-15 of the
// middle of two integers is slower for 16-bit rows, in which such quotients are common: half
// of the largest element is 63.5.)
template <uint32_t DT, int V>
VM_DEV void i8_rows(const Run<DT, 8> (&x)[V], uint32_t lph, float (&scale)[V], v2u (&q)[V]) {
  uint32_t mb[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    if constexpr (DT == DT_F32) {
      mb[k] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) mb[k] = max(mb[k], x[k].w[i] & 0x7FFFFFFFu);
    } else {
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 m = {0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = x[k].w[i] & 0x7FFF7FFFu;
        m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w));
      }
      mb[k] = max(uint32_t(m.x), uint32_t(m.y));
    }
  }
  head_max(mb, lph);
  constexpr float kRound = 12582912.0f;
  uint32_t b[V][8];
  bool rare = false;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const float mx = DT == DT_F32 ? __uint_as_float(mb[k]) : DT == DT_BF16 ? __uint_as_float(mb[k] << 16) : f16_to_f32(uint16_t(mb[k]));
    const float s = mx < INFINITY ? mx * (1.0f / 127.0f) : __builtin_nanf("");
    scale[k] = s;
    const bool plain = s >= 1e-20f && s <= 1e20f;
    const float y = plain ? 1.0f / s : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = x[k].get(i);
      float d = f * y;
      d = fmaf(fmaf(-s, d, f), y, d);
      d = fmaf(fmaf(-s, d, f), y, d);
      b[k][i] = __float_as_uint(d + kRound);
    }
    rare = rare || (s > 0.0f && !plain);
  }
  if (__any(rare)) {
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        b[k][i] = uint32_t(int32_t(fminf(fmaxf(rintf(__fdiv_rn(x[k].get(i), scale[k])), -127.0f), 127.0f)));
  }
#pragma unroll
  for (int k = 0; k < V; ++k) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo = __builtin_amdgcn_perm(b[k][4 * i + 1], b[k][4 * i], 0x0C0C0400u);
      const uint32_t hi = __builtin_amdgcn_perm(b[k][4 * i + 3], b[k][4 * i + 2], 0x04000C0Cu);
      w[i] = scale[k] > 0.0f ? lo | hi : 0;
    }
    q[k] = v2u_make(w[0], w[1]);
  }
}

// DT: the rows' element type; Q8: pages of i8 (else of DT).  READ: out of the pages.
template <uint32_t DT, bool Q8, bool READ>
VM_TILE void cache_move(Args A, uint32_t ti, uint32_t lo, uint32_t hi) {
  A = uargs(A);
  lo = uni(lo);
  hi = uni(hi);
  const VM_K Task& t = task_of(A, ti);
  const PagedDesc D = paged_desc(A, t);
  const uint32_t TB = t.p[7] & 0xFF, tid = threadIdx.x, lane = tid & 63, odt = (t.tile_op >> 8) & 0xFF;
  const VM_G int32_t* cu = gcast<int32_t>(resolve(A, t.p[3]));
  const VM_G int32_t* lens = gcast<int32_t>(resolve(A, t.p[4]));
  const VM_G int32_t* table = gcast<int32_t>(resolve(A, t.p[5]));
  // pages and rows of keys and values
  gbyte* const kpg = resolve(A, READ ? t.a : t.dst);
  gbyte* const vpg = resolve(A, READ ? t.b : t.p[0]);
  gbyte* const krw = resolve(A, READ ? t.dst : t.a);
  gbyte* const vrw = resolve(A, READ ? t.p[0] : t.b);
  VM_G float* const ksc = gcast<float>(resolve(A, t.p[1]));
  VM_G float* const vsc = gcast<float>(resolve(A, t.p[2]));
  // groups of lph lanes, a head's eight channels each: G1 (a power of two that divides the
  // heads) times G2 rows
  const uint32_t lph = pow2_at_least(D.hd / 8), l = tid & (lph - 1), grp = tid / lph;
  const uint32_t G1 = min(kBlock / lph, D.Hkv & -D.Hkv), G2 = kBlock / lph / G1, s2 = uint32_t(__builtin_ctz(G2));
  const uint32_t g1 = grp & (G1 - 1), g2 = grp / G1, hd8 = D.hd / 8, c = min(l, hd8 - 1) * 8;
  const bool on = l < hd8;
  // a wave's LDS: its rows' places, then a batch's raw runs and scales, a lane its own
  typedef Run<READ && Q8 ? DT_BF16 : DT, READ && Q8 ? 4 : 8> Raw;      // 8 bytes of i8
  constexpr uint32_t W = Raw::kWords, U = W <= 4 ? 8 : 4, V = 2;
  constexpr uint32_t kLane = (2 * U * (W + 1) + 1) * 4;                // bytes a lane
  typedef __attribute__((address_space(3))) uint32_t lds_u;
  lds_u* place = (lds_u*)(lds_ptr<uint8_t>() + uni(tid >> 6) * 64 * kLane);
  lds_u* raw = place + 64 + lane;
  lds_u* scl = raw + 2 * U * W * 64;
  for (uint32_t tile = lo; tile < hi; ++tile) {
    const uint32_t r0 = tile * TB;
    if (r0 >= D.T) break;
    // steps: J of a group's row each G2th, for each G1th head; keys and values together
    const uint32_t nr = min(TB, D.T - r0), J = (nr + G2 - 1) >> s2, steps = D.Hkv / G1 * J;
    const uint64_t ka = uint64_t(r0) * D.ars + D.aoff + c, va = uint64_t(r0) * D.brs + D.boff + c;
    struct At {
      uint32_t j, h;                     // row j G2 + g2 of the tile, head h + g1
    };
    auto next = [&](At& q) {
      const bool end = q.j + 1 == J;
      q.h = end ? q.h + G1 : q.h;
      q.j = end ? 0 : q.j + 1;
    };
    At ld{0, 0}, st{0, 0};
    Raw x[2 * U];
    float xs[2 * U];
    auto load = [&](uint32_t s) {
#pragma unroll
      for (uint32_t k = 0; k < U; ++k) {
        if (s + k >= steps) continue;
        const uint32_t r = min(ld.j * G2 + g2, nr - 1), h = ld.h + g1;
        if constexpr (READ) {
          // rows without a place read slot 0 of page 0 (not used)
          const uint32_t p = place[r], row = p == kNoPlace ? 0 : p + h * D.P;
          const uint64_t e = uint64_t(row) * D.hd + c;
          if constexpr (Q8) {
            x[2 * k].load(kpg, e / 2);
            x[2 * k + 1].load(vpg, e / 2);
            xs[2 * k] = ksc[row];
            xs[2 * k + 1] = vsc[row];
          } else {
            x[2 * k].load(kpg, e);
            x[2 * k + 1].load(vpg, e);
          }
        } else {
          x[2 * k].load(krw, ka + uint64_t(r) * D.ars + uint64_t(h) * D.ahs);
          x[2 * k + 1].load(vrw, va + uint64_t(r) * D.brs + uint64_t(h) * D.bhs);
        }
        next(ld);
      }
    };
    if (!READ) load(0);
    place[lane] = row_places(D, cu, lens, table, r0, nr);
    __builtin_amdgcn_wave_barrier();
    if (READ) load(0);
    for (uint32_t s = 0; s < steps; s += U) {
      const uint32_t n = min(U, steps - s);
#pragma unroll
      for (uint32_t k = 0; k < 2 * U; ++k) {
        if (k >= 2 * n) continue;
#pragma unroll
        for (uint32_t i = 0; i < W; ++i) raw[(k * W + i) * 64] = x[k].w[i];
        if constexpr (READ && Q8) scl[k * 64] = __float_as_uint(xs[k]);
      }
      load(s + U);
#pragma unroll 1
      for (uint32_t k0 = 0; k0 < n; k0 += V) {
        Raw o[2 * V];
        float sc[2 * V];
        uint64_t at[V];                // element of the rows (read) or the pages (append)
        uint32_t row[V];
        bool in[V], ok[V];
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) {
          const uint32_t rr = st.j * G2 + g2, r = min(rr, nr - 1), h = st.h + g1, p = place[r];
          ok[k] = p != kNoPlace;
          in[k] = rr < nr && on && k0 + k < n && (READ || ok[k]);
          row[k] = p + h * D.P;
          at[k] = (READ ? uint64_t(r0 + r) * D.Hkv + h : uint64_t(row[k])) * D.hd + c;
          const uint32_t kk = 2 * min(k0 + k, n - 1);
#pragma unroll
          for (uint32_t b = 0; b < 2; ++b) {
#pragma unroll
            for (uint32_t i = 0; i < W; ++i) o[2 * k + b].w[i] = raw[((kk + b) * W + i) * 64];
            if constexpr (READ && Q8) sc[2 * k + b] = __uint_as_float(scl[(kk + b) * 64]);
          }
          next(st);
        }
        if constexpr (READ) {
          auto put = [&](auto type) {
            typedef decltype(type) Y;
#pragma unroll
            for (uint32_t k = 0; k < 2 * V; ++k) {
              float f[8];
              if constexpr (Q8) {
                i8_get(v2u_make(o[k].w[0], o[k].w[1]), f);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] *= sc[k];
              } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = o[k].get(i);
              }
              Y y;
              y.put(f);
#pragma unroll
              for (int i = 0; i < Y::kWords; ++i) y.w[i] = ok[k / 2] ? y.w[i] : 0;
              if (in[k / 2]) y.store(k & 1 ? vrw : krw, at[k / 2]);
            }
          };
          if (odt == DT_F32) put(Run<DT_F32, 8>());
          else if (odt == DT_BF16) put(Run<DT_BF16, 8>());
          else put(Run<DT_F16, 8>());
        } else if constexpr (Q8) {
          v2u q[2 * V];
          i8_rows<DT, 2 * V>(o, lph, sc, q);
#pragma unroll
          for (uint32_t k = 0; k < 2 * V; ++k)
            if (in[k / 2]) {
              *(VM_G v2u*)((k & 1 ? vpg : kpg) + at[k / 2]) = q[k];
              if (l == 0) (k & 1 ? vsc : ksc)[row[k / 2]] = sc[k];
            }
        } else {
#pragma unroll
          for (uint32_t k = 0; k < 2 * V; ++k)
            if (in[k / 2]) o[k].store(k & 1 ? vpg : kpg, at[k / 2]);
        }
      }
    }
  }
  __syncthreads();
}

VM_DEV void cache_tiles(Args A, uint32_t ti, uint32_t lo, uint32_t hi, bool read) {
  const VM_K Task& t = task_of(A, ti);
  const VM_K int32_t* d = aux_of(A) + t.p[6];
  const uint32_t cdt = d[PD_CDT], rdt = ((t.tile_op >> (read ? 8 : 16)) & 0xFF);
  if (cdt == DT_I8) {
    if (read) cache_move<DT_F32, true, true>(A, ti, lo, hi);
    else if (rdt == DT_BF16) cache_move<DT_BF16, true, false>(A, ti, lo, hi);
    else if (rdt == DT_F16) cache_move<DT_F16, true, false>(A, ti, lo, hi);
    else cache_move<DT_F32, true, false>(A, ti, lo, hi);
  } else if (read) {
    if (cdt == DT_BF16) cache_move<DT_BF16, false, true>(A, ti, lo, hi);
    else if (cdt == DT_F16) cache_move<DT_F16, false, true>(A, ti, lo, hi);
    else cache_move<DT_F32, false, true>(A, ti, lo, hi);
  } else {
    if (cdt == DT_BF16) cache_move<DT_BF16, false, false>(A, ti, lo, hi);
    else if (cdt == DT_F16) cache_move<DT_F16, false, false>(A, ti, lo, hi);
    else cache_move<DT_F32, false, false>(A, ti, lo, hi);
  }
}

}  // namespace vm
