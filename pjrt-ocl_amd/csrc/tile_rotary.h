// TOP_ROTARY, TOP_ROTARY_GRAD (extensions): rotary positions of the heads of
// [T, H, hd] rows, with an optional RMS norm of each head in the same pass.
//
//   z[d] = x[d] r w[d],  r = 1 / sqrt(mean_d x[d]^2 + eps)       (no norm: z = x)
//   a_i  = pos[t] f_i,   y[c] = m (z[c] cos a - z[s] sin a),  y[s] = m (z[s] cos a + z[c] sin a)
//
// for the channel pairs (c, s) = (i, i + R), or (2 i, 2 i + 1) when interleaved, i < R =
// rot / 2; channels past rot pass (y = z).  The gradient: dz = R^T dy, dx = r w dz -
// x r^3 / hd sum_d w dz x, dweight[d] = sum over rows and heads of dz[d] x[d] r.
//
// Angles: a frequency comes as a 64-bit fixed-point fraction of a turn, so that pos *
// f modulo one turn is one 64-bit integer product (a far position loses nothing: in
// f32 position 10^6 would leave the fastest pair 0.06 rad off).  Its top 32 bits give
// the quadrant and, as a signed 30-bit fraction, an angle in [-pi/4, pi/4], whose
// sine and cosine are Taylor sums to x^9 and x^10 (the next terms are below 2^-28).
//
// A slot is PW channel pairs (or 2 PW channels that pass): with PW = 8 or 4 it is read and
// written in 16 / 8 byte runs.  LPH lanes (a power of two) hold a head, 64 / LPH heads go
// through a wave at a time, each lane with the same slots of every head.  A wave takes
// kRotRows rows at a time: their sines go into LDS once (a pair a lane, 35 instructions each; each
// lane working its own eight pairs out for every row took 48 of 99 us for 8192 rows of 40
// heads), then the (row, head) pairs pass in batches, the next batch's loads in flight
// while one is computed (there is one wave per SIMD to hide them).  x is read and y written
// once: 8192 rows of 40 heads of 128, bf16 with the norm, 168 MB in 48 us (3.5 TB/s), the
// gradient of 4096 rows of 32 heads, 101 MB in 39.  What is left beside HBM is instruction
// issue, some 150 instructions for a lane's 16 channels: larger batches change nothing, and
// a division less for each pair and the hardware's 1 / sqrt took 4 %.  As leaves they take 2 to
// 4 us less, but then the kernel saves more around every call: a decoder's steps took 3 % longer.
#pragma once
#include "vm_device.h"

namespace vm {

constexpr uint32_t kRotRows = 8;                           // rows of a wave's table of sines at most
constexpr uint32_t kRotTable = kRotRows * (128 + 8) * 2;   // floats per wave

struct RotDesc {
  uint32_t T, H, hd, rot, flags;
  float eps, mag;
  uint32_t ars, ahs, aoff, brs, bhs, boff;
};
VM_DEV RotDesc rot_desc(Args A, const VM_K Task& t) {
  const VM_K int32_t* d = aux_of(A) + t.p[2];
  return RotDesc{uint32_t(d[RD_T]), uint32_t(d[RD_H]), uint32_t(d[RD_HD]), uint32_t(d[RD_ROT]), uint32_t(d[RD_FLAGS]),
                 __int_as_float(d[RD_EPS]), __int_as_float(d[RD_MAG]), uint32_t(d[RD_ARS]), uint32_t(d[RD_AHS]),
                 uint32_t(d[RD_AOFF]), uint32_t(d[RD_BRS]), uint32_t(d[RD_BHS]), uint32_t(d[RD_BOFF])};
}

// 16, 8 and 4 bytes at any element's alignment
typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u1 __attribute__((aligned(2)));

// Runs of N elements as raw 32-bit words (or 16-bit halves for N = 1 of a 16-bit
// type), at any element alignment, and their f32 values.
template <uint32_t DT, int N>
struct Run {
  static constexpr int kBytes = N * (DT == DT_F32 ? 4 : 2);
  static constexpr int kWords = kBytes >= 4 ? kBytes / 4 : 1;
  uint32_t w[kWords];
  VM_DEV void load(const gbyte* base, uint64_t e) {
    const gbyte* p = base + e * (DT == DT_F32 ? 4 : 2);
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const u4 v = *(const VM_G u4*)(p + 16 * i);
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
      }
    } else if constexpr (kBytes == 8) {
      const u2 v = *(const VM_G u2*)p;
      w[0] = v.x; w[1] = v.y;
    } else if constexpr (kBytes == 4) {
      w[0] = *(const VM_G u1*)p;
    } else {
      w[0] = *(const VM_G uint16_t*)p;
    }
  }
  VM_DEV float get(int i) const {
    if constexpr (DT == DT_F32) return __uint_as_float(w[i]);
    const uint32_t h = (w[i / 2] >> (16 * (i & 1)));
    if constexpr (DT == DT_BF16) return __uint_as_float((i & 1) ? (w[i / 2] & 0xFFFF0000u) : h << 16);
    else return f16_to_f32(uint16_t(h));
  }
  VM_DEV void put(const float (&f)[N]) {
    if constexpr (DT == DT_F32) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = __float_as_uint(f[i]);
    } else if constexpr (N == 1) {
      w[0] = DT == DT_BF16 ? f32_to_bf16(f[0]) : f32_to_f16(f[0]);
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 2)
        w[i / 2] = DT == DT_BF16 ? pack_bf16x2(f[i], f[i + 1]) : f32_to_f16(f[i]) | (uint32_t(f32_to_f16(f[i + 1])) << 16);
    }
  }
  VM_DEV void store(gbyte* base, uint64_t e) const {
    gbyte* p = base + e * (DT == DT_F32 ? 4 : 2);
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) *(VM_G u4*)(p + 16 * i) = u4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
    } else if constexpr (kBytes == 8) {
      *(VM_G u2*)p = u2{w[0], w[1]};
    } else if constexpr (kBytes == 4) {
      *(VM_G u1*)p = w[0];
    } else {
      *(VM_G uint16_t*)p = uint16_t(w[0]);
    }
  }
};

// Sine and cosine of pos * f, f a 64-bit fixed-point fraction of a turn.
VM_DEV void turn_sincos(int32_t pos, uint32_t flo, uint32_t fhi, float* sn, float* cs) {
  const uint32_t top = uint32_t((uint64_t(int64_t(pos)) * ((uint64_t(fhi) << 32) | flo)) >> 32);
  const uint32_t q = (top + 0x20000000u) >> 30;                      // quadrant 0..3
  const float x = float(int32_t(top - (q << 30))) * 1.4629180792671596e-9f;   // 2 pi / 2^32
  const float x2 = x * x;
  const float s = x + x * x2 * fmaf(x2, fmaf(x2, fmaf(x2, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f);
  const float c = 1.0f + x2 * fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f),
                                            4.1666667e-2f), -0.5f);
  const float a = (q & 1) ? c : s, b = (q & 1) ? s : c;
  *sn = (q & 2) ? -a : a;
  *cs = ((q + 1) & 2) ? -b : b;
}

// Sum over the LPH (a power of two) adjacent lanes of a head, the same in each.
VM_DEV float head_sum(float x, uint32_t lph) {
  if (lph > 1) x += dpp<0xB1>(x);
  if (lph > 2) x += dpp<0x4E>(x);
  if (lph > 4) x += __shfl_xor(x, 4, 64);
  if (lph > 8) x += __shfl_xor(x, 8, 64);
  if (lph > 16) x += __shfl_xor(x, 16, 64);
  if (lph > 32) x += __shfl_xor(x, 32, 64);
  return x;
}

// 1 / sqrt(x), to an ulp; 0 and denormal x are scaled (the instruction takes them for 0).
VM_DEV float inv_sqrt(float x) {
  const bool small = x < 0x1p-120f;
  const float r = __builtin_amdgcn_rsqf(small ? x * 0x1p+24f : x);
  return small ? r * 0x1p+12f : r;
}

// The slots of a lane: NS at most (lane, lane + LPH, ...), their channels, weights and places
// in the table of sines.
template <int PW, int NS, bool INTER>
struct RotSlots {
  uint32_t c0[NS], c1[NS];         // first channels of the slot's two runs of PW
  uint32_t at[NS];                 // its first pair in a row of the table
  bool on[NS];
  float w0[NS][PW], w1[NS][PW];

  VM_DEV void place(const RotDesc& D, uint32_t l, uint32_t lph) {
    const uint32_t rs = D.rot / (2 * PW), all = D.hd / (2 * PW), R = D.rot / 2;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const uint32_t s = l + n * lph;
      on[n] = s < all;
      const bool turn = s < rs;
      const uint32_t k = min(s, all - 1);
      c0[n] = (!INTER && turn) ? k * PW : k * 2 * PW;
      c1[n] = (!INTER && turn) ? R + k * PW : k * 2 * PW + PW;
      at[n] = turn ? k * PW : R;   // past the pairs a row of the table has PW turns of 0
    }
  }
  VM_DEV void weights(const VM_G float* w) {
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < PW; ++i) {
        w0[n][i] = w[c0[n] + i];
        w1[n][i] = w[c1[n] + i];
      }
  }
  // cosine and sine (times the magnitude) of the slot's pairs in the table row
  VM_DEV void turns(const float* row, int n, float (&cs)[PW], float (&sn)[PW]) const {
    const float* p = row + 2 * at[n];
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      cs[i] = p[2 * i];
      sn[i] = p[2 * i + 1];
    }
  }
  // element i of run 0 / run 1: with interleaved slots the pair is (2 i, 2 i + 1)
  // of the slot's 2 PW contiguous channels
  template <class R>
  VM_DEV static void pair(const R& r0, const R& r1, int i, float* a, float* b) {
    if constexpr (INTER && PW > 1) {
      *a = 2 * i < PW ? r0.get((2 * i) % PW) : r1.get((2 * i) % PW);
      *b = 2 * i < PW ? r0.get((2 * i + 1) % PW) : r1.get((2 * i + 1) % PW);
    } else {
      *a = r0.get(i);
      *b = r1.get(i);
    }
  }
  VM_DEV static void unpair(float (&f0)[PW], float (&f1)[PW], int i, float a, float b) {
    if constexpr (INTER && PW > 1) {
      if (2 * i < PW) { f0[(2 * i) % PW] = a; f0[(2 * i + 1) % PW] = b; }
      else { f1[(2 * i) % PW] = a; f1[(2 * i + 1) % PW] = b; }
    } else {
      f0[i] = a;
      f1[i] = b;
    }
  }
  // the norm's weights of pair i
  VM_DEV void weight_pair(int n, int i, float* a, float* b) const {
    if constexpr (INTER && PW > 1) {
      *a = 2 * i < PW ? w0[n][(2 * i) % PW] : w1[n][(2 * i) % PW];
      *b = 2 * i < PW ? w0[n][(2 * i + 1) % PW] : w1[n][(2 * i + 1) % PW];
    } else {
      *a = w0[n][i];
      *b = w1[n][i];
    }
  }
};

// The wave's table of the turns of rows [row, row + nr): [nr][R + pw] pairs (cosine, sine)
// times the magnitude, `sign` -1 to rotate back, and pw turns of 0 at the end of a row.
VM_DEV void rot_table(const RotDesc& D, float* tab, const VM_G int32_t* pos, const VM_G uint32_t* freq, uint32_t row,
                      uint32_t nr, uint32_t pw, float sign) {
  const uint32_t lane = threadIdx.x & 63, R = D.rot / 2, ld = 2 * (R + pw);
  for (uint32_t i = lane; i < R + pw; i += 64) {
    const uint32_t k = min(i, R - 1), flo = freq[2 * k], fhi = freq[2 * k + 1];
    int32_t p[kRotRows];
#pragma unroll
    for (uint32_t r = 0; r < kRotRows; ++r) p[r] = pos[min(row + min(r, nr - 1), D.T - 1)];
#pragma unroll
    for (uint32_t r = 0; r < kRotRows; ++r) {
      if (r >= nr) break;
      float s, c;
      turn_sincos(p[r], flo, fhi, &s, &c);
      tab[r * ld + 2 * i] = i < R ? c * D.mag : 1.0f;
      tab[r * ld + 2 * i + 1] = i < R ? s * D.mag * sign : 0.0f;
    }
  }
  __builtin_amdgcn_wave_barrier();       // the wave's own LDS operations are in order
}

VM_DEV uint32_t pow2_at_least(uint32_t n) { return n <= 1 ? 1u : 1u << (32 - __builtin_clz(n - 1)); }

// A lane's (row, head) pairs p0, p0 + by, ... of rows of `nh` heads, without a division each.
// next(): row and head (past row nr - 1 of the last row), and whether it is within.
struct RotPairs {
  uint32_t r, h, dr, dh, nh;
  VM_DEV RotPairs(uint32_t p0, uint32_t by, uint32_t heads) : nh(heads) {
    r = p0 / nh;
    h = p0 - r * nh;
    dr = by / nh;
    dh = by - dr * nh;
  }
  VM_DEV bool next(uint32_t nr, uint32_t* row, uint32_t* head) {
    *row = min(r, nr - 1);
    *head = h;
    const bool in = r < nr;
    h += dh;
    r += dr;
    if (h >= nh) {
      h -= nh;
      ++r;
    }
    return in;
  }
};

// A lane's raw runs of N steps: x, or dy and then x.
template <uint32_t DT, int PW, int NS, bool GRAD = false>
struct RotBatch {
  template <int N>
  struct X {
    static constexpr int kN = N;
    Run<DT, PW> r0[N][NS], r1[N][NS];
    Run<DT, PW> x0[GRAD ? N : 1][NS], x1[GRAD ? N : 1][NS];
  };
};

// Steps 0 .. n / hpw of a wave's (row, head) pairs, 64 / LPH pairs each: whole batches of KB
// steps (no branch within, so that their chains of latencies overlap), the next one's loads
// in flight, then the rest one step at a time.  load(first step, batch), compute(first step,
// batch); before() runs once the first loads are under way.
template <template <int> class Batch, int KB, class Load, class Compute, class Before>
VM_DEV void rot_steps(uint32_t n, uint32_t hpw, Load load, Compute compute, Before before) {
  const uint32_t steps = (n + hpw - 1) / hpw, full = n / hpw / KB;
  Batch<KB> b0, b1;
  Batch<1> b;
  if (full) load(0, b0);
  else load(0, b);
  before();
  if (full) {
    for (uint32_t i = 0; i < full; i += 2) {
      if (i + 1 < full) load((i + 1) * KB, b1);
      compute(i * KB, b0);
      if (i + 1 >= full) break;
      if (i + 2 < full) load((i + 2) * KB, b0);
      compute((i + 1) * KB, b1);
    }
    if (full * KB < steps) load(full * KB, b);
  }
  for (uint32_t s = full * KB; s < steps; ++s) {
    compute(s, b);
    if (s + 1 < steps) load(s + 1, b);
  }
}

template <uint32_t DT, int PW, int NS, bool INTER>
VM_DEV void rotary_units(Args A, uint32_t ti, uint32_t lo, uint32_t hi) {
  const VM_K Task& t = task_of(A, ti);
  const RotDesc D = rot_desc(A, t);
  const uint32_t Z = t.p[3], lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const uint32_t lph = min(64u, pow2_at_least(D.hd / (2 * PW))), hpw = 64 / lph;
  const uint32_t l = lane & (lph - 1), hg = lane / lph;
  const gbyte* x = resolve(A, t.a);
  gbyte* y = resolve(A, t.dst);
  const VM_G int32_t* pos = gcast<int32_t>(resolve(A, t.p[0]));
  const VM_G uint32_t* freq = gcast<uint32_t>(resolve(A, t.p[1]));
  const bool norm = D.flags & ROT_NORM;
  const float sign = (D.flags & ROT_INVERSE) ? -1.0f : 1.0f;
  typedef Run<DT, PW> R;
  constexpr int KB = (DT == DT_F32 ? 2 : 4) / NS;               // a batch's loads: 64 bytes a lane, two in flight
  RotSlots<PW, NS, INTER> S;
  S.place(D, l, lph);
  if (norm) S.weights(gcast<float>(resolve(A, t.b)));
  const float inv_hd = 1.0f / float(D.hd);
  float* tab = lds_ptr<float>() + wave * kRotTable;
  const uint32_t ld = 2 * (D.rot / 2 + PW);
  // rows [row, row + nr), heads [h0, h1)
  auto unit = [&](uint32_t row, uint32_t nr, uint32_t h0, uint32_t h1) {
    const uint32_t nh = h1 - h0, n = nr * nh;
    RotPairs pl(hg, hpw, nh), ps = pl;
    auto load = [&](uint32_t s0, auto& B) {
#pragma unroll
      for (int k = 0; k < B.kN; ++k) {
        uint32_t r, h;
        pl.next(nr, &r, &h);
        h += h0;
        const uint64_t e = uint64_t(row + r) * D.ars + uint64_t(h) * D.ahs + D.aoff;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          B.r0[k][s].load(x, e + S.c0[s]);
          B.r1[k][s].load(x, e + S.c1[s]);
        }
      }
    };
    auto compute = [&](uint32_t s0, const auto& B) {
#pragma unroll
      for (int k = 0; k < B.kN; ++k) {
        uint32_t r, h;
        const bool in = ps.next(nr, &r, &h);
        h += h0;
        float z = 1.0f;
        if (norm) {
          float ss = 0.0f;
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int i = 0; i < PW; ++i) {
              const float a = S.on[s] ? B.r0[k][s].get(i) : 0.0f, c = S.on[s] ? B.r1[k][s].get(i) : 0.0f;
              ss = fmaf(a, a, fmaf(c, c, ss));
            }
          z = inv_sqrt(fmaf(head_sum(ss, lph), inv_hd, D.eps));
        }
        const uint64_t e = (uint64_t(row + r) * D.H + h) * D.hd;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          float f0[PW], f1[PW], cs[PW], sn[PW];
          S.turns(tab + r * ld, s, cs, sn);
#pragma unroll
          for (int i = 0; i < PW; ++i) {
            float a, c;
            S.pair(B.r0[k][s], B.r1[k][s], i, &a, &c);
            if (norm) {
              float wa, wb;
              S.weight_pair(s, i, &wa, &wb);
              a = a * z * wa;
              c = c * z * wb;
            }
            S.unpair(f0, f1, i, a * cs[i] - c * sn[i], c * cs[i] + a * sn[i]);
          }
          R o0, o1;
          o0.put(f0);
          o1.put(f1);
          if (S.on[s] && in) {
            o0.store(y, e + S.c0[s]);
            o1.store(y, e + S.c1[s]);
          }
        }
      }
    };
    rot_steps<RotBatch<DT, PW, NS>::template X, KB>(n, hpw, load, compute,
                                                    [&] { rot_table(D, tab, pos, freq, row, nr, PW, sign); });
  };
  // Z = 1: a tile is four rows, a wave takes its quarter of the entry's rows, kRotRows at a
  // time; else four (row, split) pairs, a wave every fourth
  const uint32_t n0 = 4 * lo, rows = min(D.T * Z, 4 * hi) - n0, hz = (D.H + Z - 1) / Z;   // heads of a split
  uint32_t u = n0 + (Z == 1 ? rows * wave / 4 : wave);
  const uint32_t end = Z == 1 ? n0 + rows * (wave + 1) / 4 : n0 + rows;
  while (u < end) {
    const uint32_t nr = Z == 1 ? min(kRotRows, end - u) : 1, h0 = Z == 1 ? 0 : u % Z * hz;
    if (h0 < D.H) unit(Z == 1 ? u : u / Z, nr, h0, min(D.H, h0 + hz));
    u += Z == 1 ? nr : 4;
  }
}

// Worker `tile` of p3: a contiguous share of the (row, head) pairs, a quarter of it a wave,
// with the lane's part of dweight in registers until the end; then the head groups of a
// wave and the four waves are added in LDS and left in p5, and the worker that arrives
// last adds the workers' rows into p6, all in an order of their own.
template <uint32_t DT, int PW, int NS, bool INTER>
VM_DEV void rotary_grad_worker(Args A, uint32_t ti, uint32_t tile) {
  const VM_K Task& t = task_of(A, ti);
  const RotDesc D = rot_desc(A, t);
  const uint32_t W = t.p[3], lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const uint32_t lph = min(64u, pow2_at_least(D.hd / (2 * PW))), hpw = 64 / lph;
  const uint32_t l = lane & (lph - 1), hg = lane / lph;
  const gbyte* dy = resolve(A, t.a);
  const gbyte* x = resolve(A, t.b);
  gbyte* dx = resolve(A, t.dst);
  const VM_G int32_t* pos = gcast<int32_t>(resolve(A, t.p[0]));
  const VM_G uint32_t* freq = gcast<uint32_t>(resolve(A, t.p[1]));
  typedef Run<DT, PW> R;
  constexpr int KB = DT == DT_F32 || NS > 1 ? 1 : 2;
  RotSlots<PW, NS, INTER> S;
  S.place(D, l, lph);
  S.weights(gcast<float>(resolve(A, t.p[4])));
  float g0[NS][PW], g1[NS][PW];                    // dweight of the pair's first / second channel
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int i = 0; i < PW; ++i) g0[n][i] = g1[n][i] = 0.0f;
  const float inv_hd = 1.0f / float(D.hd);
  float* tab = lds_ptr<float>() + wave * kRotTable;
  const uint32_t ld = 2 * (D.rot / 2 + PW), H = D.H;
  const uint64_t all = uint64_t(D.T) * H;
  const uint32_t t0 = uint32_t(all * tile / W), t1 = uint32_t(all * (tile + 1) / W);
  uint32_t at = t0 + uint32_t(uint64_t(t1 - t0) * wave / 4);
  const uint32_t end = t0 + uint32_t(uint64_t(t1 - t0) * (wave + 1) / 4);
  while (at < end) {
    const uint32_t row = at / H, last = uint32_t(min(uint64_t(end), uint64_t(row + kRotRows) * H));
    const uint32_t first = at - row * H, n = last - at;         // pairs `first` .. of the rows from `row`
    at = last;
    // (rows past the last pair's are the next wave's, or not there: `in` counts pairs)
    RotPairs pl(first + hg, hpw, H), ps = pl;
    const uint32_t nr = (first + n - 1) / H + 1;
    auto load = [&](uint32_t s0, auto& B) {
#pragma unroll
      for (int k = 0; k < B.kN; ++k) {
        uint32_t r, h;
        pl.next(nr, &r, &h);
        const uint64_t ye = uint64_t(row + r) * D.ars + uint64_t(h) * D.ahs + D.aoff;
        const uint64_t xe = uint64_t(row + r) * D.brs + uint64_t(h) * D.bhs + D.boff;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          B.r0[k][s].load(dy, ye + S.c0[s]);
          B.r1[k][s].load(dy, ye + S.c1[s]);
          B.x0[k][s].load(x, xe + S.c0[s]);
          B.x1[k][s].load(x, xe + S.c1[s]);
        }
      }
    };
    auto compute = [&](uint32_t s0, const auto& B) {
#pragma unroll
      for (int k = 0; k < B.kN; ++k) {
        uint32_t r, h;
        ps.next(nr, &r, &h);
        const bool in = (s0 + k) * hpw + hg < n;
        float ss = 0.0f, dot = 0.0f;
        float za[NS][PW], zb[NS][PW], xa[NS][PW], xb[NS][PW];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          float cs[PW], sn[PW];
          S.turns(tab + r * ld, s, cs, sn);
#pragma unroll
          for (int i = 0; i < PW; ++i) {
            float a, c, wa, wb;
            S.pair(B.r0[k][s], B.r1[k][s], i, &a, &c);
            S.pair(B.x0[k][s], B.x1[k][s], i, &xa[s][i], &xb[s][i]);
            xa[s][i] = S.on[s] ? xa[s][i] : 0.0f;
            xb[s][i] = S.on[s] ? xb[s][i] : 0.0f;
            S.weight_pair(s, i, &wa, &wb);
            za[s][i] = a * cs[i] - c * sn[i];
            zb[s][i] = c * cs[i] + a * sn[i];
            ss = fmaf(xa[s][i], xa[s][i], fmaf(xb[s][i], xb[s][i], ss));
            dot = fmaf(za[s][i] * wa, xa[s][i], fmaf(zb[s][i] * wb, xb[s][i], dot));
          }
        }
        const float z = inv_sqrt(fmaf(head_sum(ss, lph), inv_hd, D.eps));
        const float c = z * z * z * (head_sum(dot, lph) * inv_hd);
        const uint64_t e = (uint64_t(row + r) * H + h) * D.hd;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          float f0[PW], f1[PW];
#pragma unroll
          for (int i = 0; i < PW; ++i) {
            float wa, wb;
            S.weight_pair(s, i, &wa, &wb);
            S.unpair(f0, f1, i, z * wa * za[s][i] - xa[s][i] * c, z * wb * zb[s][i] - xb[s][i] * c);
            g0[s][i] = in ? fmaf(za[s][i] * z, xa[s][i], g0[s][i]) : g0[s][i];
            g1[s][i] = in ? fmaf(zb[s][i] * z, xb[s][i], g1[s][i]) : g1[s][i];
          }
          R o0, o1;
          o0.put(f0);
          o1.put(f1);
          if (S.on[s] && in) {
            o0.store(dx, e + S.c0[s]);
            o1.store(dx, e + S.c1[s]);
          }
        }
      }
    };
    rot_steps<RotBatch<DT, PW, NS, true>::template X, KB>(
        n, hpw, load, compute, [&] { rot_table(D, tab, pos, freq, row, min(kRotRows, D.T - row), PW, -1.0f); });
  }
  // [4 hpw][hd] partial rows in LDS: hpw * hd <= 64 * 2 PW, so at most 16 KiB.  The
  // sums are by pair: element i of g0 belongs to channel c0 + i, or c0 + 2 i interleaved
  float* lds = lds_ptr<float>();
  __syncthreads();
  float* mine = lds + (wave * hpw + hg) * D.hd;
#pragma unroll
  for (int n = 0; n < NS; ++n)
    if (S.on[n]) {
#pragma unroll
      for (int i = 0; i < PW; ++i) {
        if constexpr (INTER && PW > 1) {
          mine[S.c0[n] + 2 * i] = g0[n][i];
          mine[S.c0[n] + 2 * i + 1] = g1[n][i];
        } else {
          mine[S.c0[n] + i] = g0[n][i];
          mine[S.c1[n] + i] = g1[n][i];
        }
      }
    }
  __syncthreads();
  VM_G float* part = gcast<float>(resolve(A, t.p[5]));
  for (uint32_t d = threadIdx.x; d < D.hd; d += kBlock) {
    float s = 0.0f;
    for (uint32_t k = 0; k < 4 * hpw; ++k) s += lds[k * D.hd + d];
    part[uint64_t(tile) * D.hd + d] = s;
  }
  // the barrier orders every thread's stores (done: vmcnt 0) before thread 0's arrival, an
  // agent-scope acquire-release that writes this XCD's L2 back
  uint32_t* arrivals = reinterpret_cast<uint32_t*>(A->scratch + A->task_scratch[ti]);
  __builtin_amdgcn_s_waitcnt(0x0F70);
  __syncthreads();
  uint32_t* flag = reinterpret_cast<uint32_t*>(lds);
  if (threadIdx.x == 0) {
    const uint32_t before = __hip_atomic_fetch_add(arrivals, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    if (before == W - 1) __hip_atomic_store(arrivals, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = before == W - 1;
  }
  __syncthreads();
  const bool sum = *flag;
  __syncthreads();
  if (!sum) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  // pairs of channels by runs of rows: thread (c, run) adds rows run, run + runs, ...
  const uint32_t half = D.hd / 2, runs = kBlock / pow2_at_least(half), c = threadIdx.x % half, run = threadIdx.x / half;
  float* acc = lds;                                  // [runs][hd]
  if (run < runs) {
    float a = 0.0f, b = 0.0f;
    constexpr uint32_t U = 16;
    for (uint32_t k0 = run; k0 < W; k0 += U * runs) {
      f32x2_t v[U];
#pragma unroll
      for (uint32_t k = 0; k < U; ++k)
        v[k] = *(const VM_G f32x2_t*)(part + uint64_t(min(k0 + k * runs, W - 1)) * D.hd + 2 * c);
#pragma unroll
      for (uint32_t k = 0; k < U; ++k)
        if (k0 + k * runs < W) {
          a += v[k].x;
          b += v[k].y;
        }
    }
    acc[run * D.hd + 2 * c] = a;
    acc[run * D.hd + 2 * c + 1] = b;
  }
  __syncthreads();
  VM_G float* dw = gcast<float>(resolve(A, t.p[6]));
  for (uint32_t d = threadIdx.x; d < D.hd; d += kBlock) {
    float s = 0.0f;
    for (uint32_t k = 0; k < runs; ++k) s += acc[k * D.hd + d];
    dw[d] = s;
  }
}

template <uint32_t DT, int PW, int NS, bool INTER>
VM_TILE void rotary_run(Args A, uint32_t ti, uint32_t lo, uint32_t hi, bool grad) {
  A = uargs(A);
  lo = uni(lo);
  hi = uni(hi);
  if (!grad) {
    rotary_units<DT, PW, NS, INTER>(A, ti, lo, hi);
    return;
  }
  for (uint32_t tile = lo; tile < hi; ++tile) {
    rotary_grad_worker<DT, PW, NS, INTER>(A, ti, tile);
    __syncthreads();
  }
}

template <uint32_t DT>
VM_DEV void rotary_dispatch(Args A, uint32_t ti, uint32_t lo, uint32_t hi, bool grad) {
  const VM_K Task& t = task_of(A, ti);
  const VM_K int32_t* d = aux_of(A) + t.p[2];
  const uint32_t hd = d[RD_HD], rot = d[RD_ROT];
  const bool inter = d[RD_FLAGS] & ROT_INTERLEAVED;
  // runs of 8 channels where head and rotated part are whole slots of 16, else of 4,
  // else single pairs (two slots of up to 128 pairs a lane)
  const int pw = (hd % 16 == 0 && rot % 16 == 0) ? 8 : (hd % 8 == 0 && rot % 8 == 0) ? 4 : 1;
  if (inter) {
    if (pw == 8) rotary_run<DT, 8, 1, true>(A, ti, lo, hi, grad);
    else if (pw == 4) rotary_run<DT, 4, 1, true>(A, ti, lo, hi, grad);
    else rotary_run<DT, 1, 2, true>(A, ti, lo, hi, grad);
  } else {
    if (pw == 8) rotary_run<DT, 8, 1, false>(A, ti, lo, hi, grad);
    else if (pw == 4) rotary_run<DT, 4, 1, false>(A, ti, lo, hi, grad);
    else rotary_run<DT, 1, 2, false>(A, ti, lo, hi, grad);
  }
}

VM_DEV void rotary_tiles(Args A, uint32_t ti, uint32_t lo, uint32_t hi, bool grad) {
  const uint32_t dt = (task_of(A, ti).tile_op >> 8) & 0xFF;
  if (dt == DT_BF16) rotary_dispatch<DT_BF16>(A, ti, lo, hi, grad);
  else if (dt == DT_F16) rotary_dispatch<DT_F16>(A, ti, lo, hi, grad);
  else rotary_dispatch<DT_F32>(A, ti, lo, hi, grad);
}

}  // namespace vm
