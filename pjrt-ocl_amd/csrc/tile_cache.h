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
// A tile is p7 & 255 rows (64 at most), keys and values of every head.  Each lane of a
// wave first looks one row's place up (sequence by counting cu entries 64 at a time,
// then its length, then its page: three dependent reads for all rows together), the
// places are kept in LDS, and then groups of LPH lanes, 8 channels each, move the
// tile's (row, k or v, head) rows.  Bound by HBM; short tiles by those reads' latency.
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

constexpr uint64_t kNoPlace = ~uint64_t(0);

// Place of row r (each lane its own): page and slot in the halves, or kNoPlace.  Every lane of the
// wave calls it.
VM_DEV uint64_t row_place(const PagedDesc& D, const VM_G int32_t* cu, const VM_G int32_t* lens,
                          const VM_G int32_t* table, uint32_t r) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t s = 0;
  for (uint32_t i0 = 0; i0 < D.B; i0 += 64) {
    const uint32_t nb = min(64u, D.B - i0);
    const int32_t mine = cu[1 + i0 + min(lane, nb - 1)];
    for (uint32_t i = 0; i < nb; ++i) s += __builtin_amdgcn_readlane(mine, i) <= int32_t(r) ? 1u : 0u;
  }
  if (r >= D.T || s >= D.B) return kNoPlace;
  const int32_t c0 = cu[s], c1 = cu[s + 1], len = lens[s];
  if (c0 < 0 || c0 > int32_t(r) || c1 <= int32_t(r) || uint32_t(c1) > D.T) return kNoPlace;
  const uint32_t cap = D.MP * D.P;
  if (len < c1 - c0 || uint32_t(len) > cap) return kNoPlace;
  const uint32_t p = uint32_t(len) - (uint32_t(c1) - r);
  const uint32_t e = D.dp.quo(p);
  const int32_t page = table[uint64_t(s) * D.MP + e];
  if (page < 0 || uint32_t(page) >= D.N) return kNoPlace;
  return (uint64_t(page) << 32) | (p - e * D.P);
}

// Eight signed bytes as f32 and back.
VM_DEV void i8_get(v2u w, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = float(int32_t((i < 4 ? w.x : w.y) << (24 - 8 * (i & 3))) >> 24);
}
VM_DEV v2u i8_put(const int32_t (&q)[8]) {
  v2u w = v2u_make(0, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w.x |= (uint32_t(q[i]) & 0xFF) << (8 * i);
    w.y |= (uint32_t(q[i + 4]) & 0xFF) << (8 * i);
  }
  return w;
}

// DT: the rows' element type; Q8: pages of i8 (else of DT).  `read`: out of the pages.
template <uint32_t DT, bool Q8, bool READ>
VM_TILE void cache_move(Args A, uint32_t ti, uint32_t lo, uint32_t hi) {
  A = uargs(A);
  lo = uni(lo);
  hi = uni(hi);
  const VM_K Task& t = task_of(A, ti);
  const PagedDesc D = paged_desc(A, t);
  const uint32_t TB = t.p[7] & 0xFF, tid = threadIdx.x;
  const VM_G int32_t* cu = gcast<int32_t>(resolve(A, t.p[3]));
  const VM_G int32_t* lens = gcast<int32_t>(resolve(A, t.p[4]));
  const VM_G int32_t* table = gcast<int32_t>(resolve(A, t.p[5]));
  // pages and rows of keys (0) and values (1)
  gbyte* pg[2] = {resolve(A, READ ? t.a : t.dst), resolve(A, READ ? t.b : t.p[0])};
  gbyte* rw[2] = {resolve(A, READ ? t.dst : t.a), resolve(A, READ ? t.p[0] : t.b)};
  VM_G float* sc[2] = {gcast<float>(resolve(A, t.p[1])), gcast<float>(resolve(A, t.p[2]))};
  const uint32_t lph = pow2_at_least(D.hd / 8), l = tid & (lph - 1), grp = tid / lph, ngrp = kBlock / lph;
  const bool on = l < D.hd / 8;
  const uint32_t c = min(l, D.hd / 8 - 1) * 8;
  uint64_t* place = lds_ptr<uint64_t>();
  typedef Run<DT, 8> R;
  for (uint32_t tile = lo; tile < hi; ++tile) {
    const uint32_t r0 = tile * TB, nr = min(TB, D.T - min(D.T, r0));
    __syncthreads();
    if (tid < 64) {
      const uint64_t p = row_place(D, cu, lens, table, r0 + min(tid, TB - 1));
      if (tid < TB) place[tid] = p;
    }
    __syncthreads();
    const uint32_t total = nr * 2 * D.Hkv;
    // a fixed number of rows in flight per group
    constexpr uint32_t U = 4;
    for (uint32_t u0 = 0; u0 < total; u0 += ngrp * U) {
      R x[U];
      v2u q8[U];
      float s8[U];
      uint64_t at[U], row[U];
      uint32_t kv[U], h[U];
      bool ok[U];
#pragma unroll
      for (uint32_t k = 0; k < U; ++k) {
        const uint32_t u = u0 + k * ngrp + grp, uu = min(u, total - 1);
        const uint32_t r = uu / (2 * D.Hkv), m = uu % (2 * D.Hkv);
        kv[k] = m >= D.Hkv;
        h[k] = kv[k] ? m - D.Hkv : m;
        const uint64_t p = place[r];
        ok[k] = u < total && p != kNoPlace;
        const uint64_t pp = p == kNoPlace ? 0 : p;
        // element of the pages [N, heads, P, hd]; scales [N, heads, P] share the row index
        at[k] = (uint64_t(uint32_t(pp >> 32)) * D.Hkv + h[k]) * D.P + uint32_t(pp);
        row[k] = READ ? (uint64_t(r0 + r) * D.Hkv + h[k]) * D.hd
                      : kv[k] ? uint64_t(r0 + r) * D.brs + uint64_t(h[k]) * D.bhs + D.boff
                              : uint64_t(r0 + r) * D.ars + uint64_t(h[k]) * D.ahs + D.aoff;
        if constexpr (READ) {
          // rows without a place read slot 0 of page 0 (not used)
          if constexpr (Q8) {
            q8[k] = *(const VM_G v2u*)(pg[kv[k]] + at[k] * D.hd + c);
            s8[k] = sc[kv[k]][at[k]];
          } else {
            x[k].load(pg[kv[k]], at[k] * D.hd + c);
          }
        } else {
          x[k].load(rw[kv[k]], row[k] + c);
        }
      }
#pragma unroll
      for (uint32_t k = 0; k < U; ++k) {
        const uint32_t u = u0 + k * ngrp + grp;
        if constexpr (READ) {
          float f[8];
          if constexpr (Q8) {
            i8_get(q8[k], f);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] *= s8[k];
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = x[k].get(i);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = ok[k] ? f[i] : 0.0f;
          if (u < total && on) {
            const uint32_t odt = (t.tile_op >> 8) & 0xFF;     // the output's type, which Q8 alone lets differ
            if (odt == DT_F32) {
              Run<DT_F32, 8> o;
              o.put(f);
              o.store(rw[kv[k]], row[k] + c);
            } else if (odt == DT_BF16) {
              Run<DT_BF16, 8> o;
              o.put(f);
              o.store(rw[kv[k]], row[k] + c);
            } else {
              Run<DT_F16, 8> o;
              o.put(f);
              o.store(rw[kv[k]], row[k] + c);
            }
          }
        } else if constexpr (Q8) {
          float f[8], mx = 0.0f;
          bool fin = true;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            f[i] = x[k].get(i);
            mx = fmaxf(mx, fabsf(f[i]));
            fin = fin && fabsf(f[i]) < INFINITY;              // false for NaN too
          }
          mx = fin ? mx : INFINITY;
          for (uint32_t msk = lph >> 1; msk >= 1; msk >>= 1) mx = fmaxf(mx, __shfl_xor(mx, msk, 64));
          const float s = mx < INFINITY ? mx * (1.0f / 127.0f) : __builtin_nanf("");
          int32_t q[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float d = s > 0.0f ? rintf(__fdiv_rn(f[i], s)) : 0.0f;
            q[i] = int32_t(fminf(fmaxf(d, -127.0f), 127.0f));
          }
          if (ok[k] && on) *(VM_G v2u*)(pg[kv[k]] + at[k] * D.hd + c) = i8_put(q);
          if (ok[k] && l == 0) sc[kv[k]][at[k]] = s;
        } else {
          if (ok[k] && on) x[k].store(pg[kv[k]], at[k] * D.hd + c);
        }
      }
    }
  }
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
