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
// A slot is PW channel pairs (or 2 PW channels that pass): with PW = 8 or 4 it is read
// and written in 16 / 8 byte runs.  A wave takes one row and the heads of one of
// its p3 splits: LPH lanes a head (a power of two), 64 / LPH heads at a time, each lane
// the same slots of every head, so a lane works its sines out once per row.  Both
// are bound by HBM: x is read and y written once.
#pragma once
#include "vm_device.h"

namespace vm {

constexpr uint32_t kRotHeads = 4;      // head groups whose loads a wave has in flight at once

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

// The slots of a lane: NS at most (lane, lane + LPH, ...), their channels and sines.
template <int PW, int NS, bool INTER>
struct RotSlots {
  uint32_t c0[NS], c1[NS];         // first channels of the slot's two runs of PW
  bool on[NS];
  float sn[NS][PW], cs[NS][PW], w0[NS][PW], w1[NS][PW];

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
  // slots that pass get the angle 0 and the magnitude 1; `sign` -1 rotates back
  VM_DEV void angles(const RotDesc& D, const VM_G uint32_t* freq, int32_t pos, uint32_t l, uint32_t lph, float sign) {
    const uint32_t rs = D.rot / (2 * PW);
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const uint32_t s = l + n * lph;
#pragma unroll
      for (int i = 0; i < PW; ++i) {
        const uint32_t k = 2 * min(s * PW + i, D.rot / 2 - 1);
        float a, b;
        turn_sincos(pos, freq[k], freq[k + 1], &a, &b);
        sn[n][i] = s < rs ? a * D.mag * sign : 0.0f;
        cs[n][i] = s < rs ? b * D.mag : 1.0f;
      }
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

VM_DEV uint32_t pow2_at_least(uint32_t n) { return n <= 1 ? 1u : 1u << (32 - __builtin_clz(n - 1)); }

template <uint32_t DT, int PW, int NS, bool INTER>
VM_DEV void rotary_units(Args A, uint32_t ti, uint32_t lo, uint32_t hi) {
  const VM_K Task& t = task_of(A, ti);
  const RotDesc D = rot_desc(A, t);
  const uint32_t Z = t.p[3], lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const uint32_t lph = min(64u, pow2_at_least(D.hd / (2 * PW))), hpw = 64 / lph;
  const uint32_t l = lane & (lph - 1), hg = lane / lph;
  const uint32_t hz = (D.H + Z - 1) / Z;                        // heads of a split
  const gbyte* x = resolve(A, t.a);
  gbyte* y = resolve(A, t.dst);
  const VM_G int32_t* pos = gcast<int32_t>(resolve(A, t.p[0]));
  const VM_G uint32_t* freq = gcast<uint32_t>(resolve(A, t.p[1]));
  const bool norm = D.flags & ROT_NORM;
  const float sign = (D.flags & ROT_INVERSE) ? -1.0f : 1.0f;
  typedef Run<DT, PW> R;
  RotSlots<PW, NS, INTER> S;
  S.place(D, l, lph);
  if (norm) S.weights(gcast<float>(resolve(A, t.b)));
  const float inv_hd = 1.0f / float(D.hd);
  for (uint32_t tile = lo; tile < hi; ++tile) {
    const uint32_t u = 4 * tile + wave;
    if (u >= D.T * Z) break;
    const uint32_t row = u / Z, h0 = (u % Z) * hz, h1 = min(D.H, h0 + hz);
    if (h0 >= h1) continue;
    S.angles(D, freq, pos[row], l, lph, sign);
    const uint64_t xr = uint64_t(row) * D.ars + D.aoff, yr = uint64_t(row) * D.H * D.hd;
    for (uint32_t hb = h0; hb < h1; hb += hpw * kRotHeads) {
      R r0[kRotHeads][NS], r1[kRotHeads][NS];
#pragma unroll
      for (uint32_t k = 0; k < kRotHeads; ++k)
        if (hb + k * hpw < h1) {
          const uint32_t h = min(hb + k * hpw + hg, h1 - 1);
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            r0[k][n].load(x, xr + uint64_t(h) * D.ahs + S.c0[n]);
            r1[k][n].load(x, xr + uint64_t(h) * D.ahs + S.c1[n]);
          }
        }
#pragma unroll
      for (uint32_t k = 0; k < kRotHeads; ++k) {
        if (hb + k * hpw >= h1) break;
        const uint32_t h = hb + k * hpw + hg;
        float r = 1.0f;
        if (norm) {
          float ss = 0.0f;
#pragma unroll
          for (int n = 0; n < NS; ++n)
            if (S.on[n])
#pragma unroll
              for (int i = 0; i < PW; ++i) {
                const float a = r0[k][n].get(i), b = r1[k][n].get(i);
                ss = fmaf(a, a, fmaf(b, b, ss));
              }
          r = 1.0f / sqrtf(fmaf(head_sum(ss, lph), inv_hd, D.eps));
        }
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          float f0[PW], f1[PW];
#pragma unroll
          for (int i = 0; i < PW; ++i) {
            float a, b;
            S.pair(r0[k][n], r1[k][n], i, &a, &b);
            if (norm) {
              float wa, wb;
              S.weight_pair(n, i, &wa, &wb);
              a = a * r * wa;
              b = b * r * wb;
            }
            S.unpair(f0, f1, i, a * S.cs[n][i] - b * S.sn[n][i], b * S.cs[n][i] + a * S.sn[n][i]);
          }
          if (S.on[n] && h < h1) {
            R o0, o1;
            o0.put(f0);
            o1.put(f1);
            o0.store(y, yr + uint64_t(h) * D.hd + S.c0[n]);
            o1.store(y, yr + uint64_t(h) * D.hd + S.c1[n]);
          }
        }
      }
    }
  }
}

// Worker `tile` of p3: rows and heads in (row, head group) order, a contiguous share
// of them, with the lane's part of dweight in registers until the end; then the head
// groups of a wave and the four waves are added in LDS, in a fixed order.
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
  RotSlots<PW, NS, INTER> S;
  S.place(D, l, lph);
  S.weights(gcast<float>(resolve(A, t.p[4])));
  float g0[NS][PW], g1[NS][PW];                    // dweight of run 0 / run 1
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int i = 0; i < PW; ++i) g0[n][i] = g1[n][i] = 0.0f;
  const float inv_hd = 1.0f / float(D.hd);
  // rows [t0, t1) of the worker, its waves every fourth
  const uint32_t t0 = uint32_t(uint64_t(D.T) * D.H * tile / W), t1 = uint32_t(uint64_t(D.T) * D.H * (tile + 1) / W);
  // (row, head) pairs t0 .. t1 - 1: the waves take runs of them that share a row
  uint32_t at = t0, turn = 0;
  while (at < t1) {
    const uint32_t row = at / D.H, h0 = at % D.H, h1 = min(D.H, h0 + (t1 - at));
    at += h1 - h0;
    // a row's heads go to the waves in blocks of hpw * 2
    const uint32_t blk = hpw * 2, nblk = (h1 - h0 + blk - 1) / blk;
    bool have = false;
    for (uint32_t b = 0; b < nblk; ++b, turn = (turn + 1) & 3) {
      if (turn != wave) continue;
      if (!have) S.angles(D, freq, pos[row], l, lph, -1.0f);
      have = true;
      R y0[2][NS], y1[2][NS], x0[2][NS], x1[2][NS];
#pragma unroll
      for (uint32_t k = 0; k < 2; ++k) {
        const uint32_t h = min(h0 + b * blk + k * hpw + hg, h1 - 1);
        const uint64_t ye = uint64_t(row) * D.ars + uint64_t(h) * D.ahs + D.aoff;
        const uint64_t xe = uint64_t(row) * D.brs + uint64_t(h) * D.bhs + D.boff;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          y0[k][n].load(dy, ye + S.c0[n]);
          y1[k][n].load(dy, ye + S.c1[n]);
          x0[k][n].load(x, xe + S.c0[n]);
          x1[k][n].load(x, xe + S.c1[n]);
        }
      }
#pragma unroll
      for (uint32_t k = 0; k < 2; ++k) {
        const uint32_t h = h0 + b * blk + k * hpw + hg;
        const bool in = h < h1;
        float ss = 0.0f, dot = 0.0f;
        float za[NS][PW], zb[NS][PW], xa[NS][PW], xb[NS][PW];
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int i = 0; i < PW; ++i) {
            float a, b2, wa, wb;
            S.pair(y0[k][n], y1[k][n], i, &a, &b2);
            S.pair(x0[k][n], x1[k][n], i, &xa[n][i], &xb[n][i]);
            S.weight_pair(n, i, &wa, &wb);
            za[n][i] = a * S.cs[n][i] - b2 * S.sn[n][i];
            zb[n][i] = b2 * S.cs[n][i] + a * S.sn[n][i];
            if (S.on[n]) {
              ss = fmaf(xa[n][i], xa[n][i], fmaf(xb[n][i], xb[n][i], ss));
              dot = fmaf(za[n][i] * wa, xa[n][i], fmaf(zb[n][i] * wb, xb[n][i], dot));
            }
          }
        const float r = 1.0f / sqrtf(fmaf(head_sum(ss, lph), inv_hd, D.eps));
        const float c = r * r * r * (head_sum(dot, lph) * inv_hd);
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          float f0[PW], f1[PW];
#pragma unroll
          for (int i = 0; i < PW; ++i) {
            float wa, wb;
            S.weight_pair(n, i, &wa, &wb);
            S.unpair(f0, f1, i, r * wa * za[n][i] - xa[n][i] * c, r * wb * zb[n][i] - xb[n][i] * c);
            if (in) {
              g0[n][i] = fmaf(za[n][i] * r, xa[n][i], g0[n][i]);
              g1[n][i] = fmaf(zb[n][i] * r, xb[n][i], g1[n][i]);
            }
          }
          if (S.on[n] && in) {
            R o0, o1;
            o0.put(f0);
            o1.put(f1);
            const uint64_t e = (uint64_t(row) * D.H + h) * D.hd;
            o0.store(dx, e + S.c0[n]);
            o1.store(dx, e + S.c1[n]);
          }
        }
      }
    }
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
  VM_G float* part = gcast<float>(resolve(A, t.p[5])) + uint64_t(tile) * D.hd;
  for (uint32_t d = threadIdx.x; d < D.hd; d += kBlock) {
    float s = 0.0f;
    for (uint32_t k = 0; k < 4 * hpw; ++k) s += lds[k * D.hd + d];
    part[d] = s;
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
