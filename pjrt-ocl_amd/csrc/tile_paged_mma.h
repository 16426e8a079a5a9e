// TOP_PAGED_ATTN on the matrix cores: 16-bit queries over pages of their type or of i8,
// head sizes up to 128 (multiples of 8, of 16 for i8), run as 64 or 128: q is padded with
// zeros, and the LDS chunks past a shorter row of K or V hold that row's last one, whose
// products are 0 or are not stored.  The rows of a block are its (token, query head of the group) pairs, so K and V
// of a kv head are read once for all of its query heads.
//
// Products as in tile_attn.h: S^T (keys x 32 rows) = K Q^T and O^T (hd x 32 rows) +=
// V^T P^T, so that the S^T accumulators are already the second product's B operand, and
// keys of a 32-key half are read in kperm's order.  K and V go from the pages straight into
// LDS (global_load_lds_dwordx4), each 16-byte chunk of a key row to a swizzled slot; the
// row of a position comes from its table entry, one position a lane, handed to the lanes
// that fetch it.
//
// Two forms:
// - up to 64 rows (single tokens, short chunks; bound by HBM): the four waves take 32-key
//   blocks in turn, each through LDS stages of its own with no barrier between them, and
//   are joined at the end of the piece (paged_block_wave; up to 16 rows paged_block_few);
// - more (chunks; bound by the matrix cores): 32 U rows a wave, all waves on the same
//   64-key blocks, double-buffered with one barrier a block (paged_block_rows).
// Measured: 64 single tokens of 32 / 8 heads of 128 over 2000 to 6000 keys 228 us (4.56 TB/s of
// cache), 48 over 4000 to 12000 keys of i8 202 us (4.0 TB/s); 2048 rows over 8192 keys 321 us
// (750 TFLOP/s).
//
// i8 pages: a fragment's bytes b become the exact values b + 128 in bf16 (three
// instructions per two) and the products are corrected by 128 times the row's sum of
// q, or of the rounded P; with f16 queries K becomes exact f16.  A key's scale multiplies
// its score, a value's scale its probability before that is rounded to bf16 (f16 would
// not hold the scales' range).
//
// P is rounded to the type of the second product (bf16 / f16: half a step, 2^-8 / 2^-11
// of each weight, the row sum taken over the rounded weights); everything else is f32.  With
// f16 queries over i8 pages P is the sum of two bf16 numbers (2^-16) and the second product
// is done twice, since one bf16 would cost the output eight times its own rounding (a chunk of
// 2048 rows over 8192 keys 546 us, with bf16 queries and one product 447; 256-row blocks spill
// a little there, 276 B a lane, and 128-row ones take 659).
//
// Positions that a row does not see weigh 0, and those outside the piece or without a page
// are zeros in LDS.  A position that one row of the block sees and another does not may
// hold an infinity or NaN, and 0 times that is NaN: a block whose result is not finite is
// computed again by the general form, which leaves such positions out.
#pragma once
#include "tile_paged.h"

namespace vm {

typedef __attribute__((address_space(3))) uint32_t lds_u32;
typedef __attribute__((address_space(3))) v4u lds_v4u_t;
typedef __attribute__((address_space(3))) v4f lds_v4f_t;
typedef __attribute__((address_space(3))) v2u lds_v2u_t;
typedef int v2i_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i_t lds_v2i_t;

// 16 / 4 bytes from each lane's own address to LDS byte `lds` + 16 / 4 times the lane
// (M0 is saved and restored as in dma16).
VM_DEV void dma16_at(const gbyte* p, uint32_t lds) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %2, off\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(lds), "v"(p)
      : "memory");
}
VM_DEV void dma4_at(const gbyte* p, uint32_t lds) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dword %2, off\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(lds), "v"(p)
      : "memory");
}
template <uint32_t N>
VM_DEV void wait_vm() {
  static_assert(N < 64, "vmcnt has six bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0F70);
}

// Slots of the 16-byte chunks of key row r (chunk c at slot c ^ swz).  16-bit rows: as
// tile_attn.h, with bit 4 (K) and bit 3 (V) of the row folded in for the 16-row form,
// whose groups of 16 lanes read rows 0-3, 8-11, 16-19 and 24-27.  i8 rows (HD bytes): K
// fragments are 8-byte reads of 16 or 32 rows, V fragments transposed reads of 8 rows x 16
// or 32 channels, each spread over the banks.
template <int HD, bool Q8>
VM_DEV uint32_t pkswz(uint32_t r) {
  if constexpr (!Q8) return kswz<HD>(r) ^ ((r >> 4) & 1);
  else return HD == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
}
template <int HD, bool Q8>
VM_DEV uint32_t pvswz(uint32_t r) {
  if constexpr (!Q8) return vswz<HD>(r) ^ (((r >> 3) & 1) << 1);
  else return HD == 128 ? ((r >> 1) & 3) << 1 : ((r >> 2) & 1) << 1;
}

// Eight signed bytes as a bf16 fragment of b + 128 or an f16 one of b.
template <bool BF16>
VM_DEV u16x8 i8_frag(v2u w) {
  w.x ^= 0x80808080u;
  w.y ^= 0x80808080u;
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t s = (i < 2 ? w.x : w.y) >> (16 * (i & 1));
    if constexpr (BF16) {
      o[i] = pack_bf16x2(float(s & 0xFF), float((s >> 8) & 0xFF));
    } else {
      // 0x6400 | u is 1024 + u
      const uint32_t h = __builtin_amdgcn_perm(0x64646464u, i < 2 ? w.x : w.y, (i & 1) ? 0x04030402u : 0x04010400u);
      const f16x2_t v = __builtin_bit_cast(f16x2_t, h) + f16x2_t{_Float16(-1152.0f), _Float16(-1152.0f)};
      o[i] = __builtin_bit_cast(uint32_t, v);
    }
  }
  return __builtin_bit_cast(u16x8, v4u_make(o[0], o[1], o[2], o[3]));
}

// Sum of a q fragment's eight values.
template <bool BF16>
VM_DEV float frag_sum(const u16x8& f) {
  const v4u w = __builtin_bit_cast(v4u, f);
  return dot2_ones<BF16>(w.w, dot2_ones<BF16>(w.z, dot2_ones<BF16>(w.y, dot2_ones<BF16>(w.x, 0.0f))));
}

// A fragment of P, in two parts where one bf16 is not enough.
template <bool TWO>
struct PFrag {
  u16x8 hi;
};
template <>
struct PFrag<true> {
  u16x8 hi, lo;
};
// Eight weights as a fragment; returns the sum of what it holds.
template <bool PBF, bool TWO>
VM_DEV float pack_p(const float (&e)[8], PFrag<TWO>& f) {
  const v4u w = v4u_make(pack_h2<PBF>(e[0], e[1]), pack_h2<PBF>(e[2], e[3]), pack_h2<PBF>(e[4], e[5]), pack_h2<PBF>(e[6], e[7]));
  f.hi = __builtin_bit_cast(u16x8, w);
  float sum = frag_sum<PBF>(f.hi);
  if constexpr (TWO) {
    float d[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = e[i] - __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    PFrag<false> lo;
    sum += pack_p<PBF>(d, lo);
    f.lo = lo.hi;
  }
  return sum;
}

// What both forms share: a block's rows, its keys' rows in the pages, and the products of
// one 32-key half.
template <int HD, bool BF16, bool Q8, int U>
struct PagedMma {
  static constexpr int KS = HD / 16, DB = HD / 32;
  static constexpr uint32_t kES = Q8 ? 1 : 2;
  static constexpr uint32_t kRow = HD * kES;                   // LDS bytes of a key row
  static constexpr bool PBF = BF16 || Q8;                      // type of the second product
  static constexpr bool P2 = !BF16 && Q8;
  typedef PFrag<P2> Pf;
  VM_DEV static f32x16 pv_mma(const u16x8& v, const Pf& p, f32x16 o) {
    o = mfma16<PBF>(v, p.hi, o);
    if constexpr (P2) o = mfma16<PBF>(v, p.lo, o);
    return o;
  }

  const PagedDesc& D;
  const PagedJob& J;
  const gbyte *kp, *vp;
  const VM_G float *ksc, *vsc;
  const VM_G int32_t* table;
  DivU32 dp, dg;                       // by positions per page, by the group
  uint32_t lane, g, hd, grow, G, R;    // G: heads of the group, R: rows
  float sl2;
  u16x8 qf[U][KS];
  float qs[U];                         // 128 times the row's sum of q (bf16 over i8)
  int32_t pos[U];                      // this lane's rows' positions
  f32x16 o[U][DB];
  float m[U], l[U], pv[U];             // reference or running maximum, sums of P and of rounded P vs
  lds_u8* L;

  VM_DEV PagedMma(Args A, const VM_K Task& t, const PagedDesc& d, const PagedJob& j) : D(d), J(j) {
    kp = resolve(A, t.b);
    vp = resolve(A, t.p[0]);
    ksc = gcast<float>(resolve(A, t.p[1]));
    vsc = gcast<float>(resolve(A, t.p[2]));
    table = gcast<int32_t>(resolve(A, t.p[5])) + uint64_t(J.seq) * D.MP;
    dp = D.dp;
    dg = D.dg;
    G = dg.d;
    R = J.tokens * G;
    lane = threadIdx.x & 63;
    g = lane >> 5;
    hd = D.hd;
    grow = hd * kES;
    sl2 = D.scale * 1.4426950408889634f;
    L = (lds_u8*)uintptr_t(uni(uint32_t(reinterpret_cast<uintptr_t>(lds_ptr<lds_u8>()))));
  }
  // rows first .. first + 32 U - 1 of the block; those past R re-read the last (not stored)
  VM_DEV void load_rows(Args A, const VM_K Task& t, uint32_t first) {
    const gbyte* q = resolve(A, t.a);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = min(first + 32 * u + (lane & 31), R - 1), tok = dg.quo(i), h = J.head * G + i - tok * G;
      const uint64_t e = uint64_t(J.row0 + tok) * D.ars + uint64_t(h) * D.ahs + D.aoff;
      pos[u] = int32_t(J.pos0 + tok);
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        u16x8 f = u16x8{};
        if (16 * k + 8 * g < hd) {
          const u4 w = *(const VM_G u4*)(q + 2 * (e + 16 * k + 8 * g));
          f = __builtin_bit_cast(u16x8, v4u_make(w.x, w.y, w.z, w.w));
        }
        qf[u][k] = f;
        if constexpr (Q8 && BF16) s += frag_sum<true>(f);
      }
      if constexpr (Q8 && BF16) qs[u] = 128.0f * (s + xor32(s));
    }
    clear();
  }
  VM_DEV void clear() {
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int db = 0; db < DB; ++db) o[u][db] = f32x16{};
      m[u] = -INFINITY;
      l[u] = pv[u] = 0.0f;
    }
  }
  // table entry index of a position of the piece
  VM_DEV uint32_t entry(uint32_t key) const { return dp.quo(min(key, J.k1 - 1)); }
  // pages' row of a position whose entry is `page`, and whether it is there
  VM_DEV uint32_t page_row(uint32_t key, int32_t page, bool* ok) const {
    *ok = key < J.k1 && page >= 0 && uint32_t(page) < D.N;
    return *ok ? (uint32_t(page) * D.Hkv + J.head) * D.P + (key - dp.quo(key) * D.P) : 0u;
  }
  // S^T of keys 32 half .. + 31 of the K block at LDS byte `k`
  VM_DEV void scores(const lds_u8* k, int u, f32x16& s, const u16x8 (&kf)[KS]) {
    s = f32x16{};
#pragma unroll
    for (int st = 0; st < KS; ++st) s = mfma16<BF16>(kf[st], qf[u][st], s);
  }
  VM_DEV void k_frags(const lds_u8* k, u16x8 (&kf)[KS]) {
    const uint32_t r = kperm(lane & 31), sw = pkswz<HD, Q8>(r);
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      if constexpr (Q8)
        kf[st] = i8_frag<BF16>(*(const lds_v2u_t*)(k + r * kRow + ((uint32_t(st) ^ sw) * 16) + 8 * g));
      else
        kf[st] = *(const lds_u16x8*)(k + r * kRow + (((2 * uint32_t(st) + g) ^ sw) * 16));
    }
  }
  // V^T fragments of keys 16 ks .. + 15 of the V block at LDS byte `v`
  VM_DEV void v_frags(const lds_u8* v, int ks, u16x8 (&vf)[DB]) {
    const uint32_t gq = lane >> 4;
    if constexpr (Q8) {
      const uint32_t e = (lane & 15) >> 1, q = lane & 1, row = 8 * (gq >> 1) + e, sw = pvswz<HD, Q8>(row);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const v2i_t w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (lds_v2i_t*)(v + (16 * ks + row) * kRow + (((2 * uint32_t(db) + (gq & 1)) ^ sw) * 16) + 8 * q));
        vf[db] = i8_frag<true>(v2u_make(uint32_t(w.x), uint32_t(w.y)));
      }
    } else {
      const uint32_t e = (lane >> 2) & 3, q = lane & 3, row = 8 * (gq >> 1) + e, sw = pvswz<HD, Q8>(row);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const lds_u8* p = v + (16 * ks + row) * kRow + (((4 * uint32_t(db) + 2 * (gq & 1) + (q >> 1)) ^ sw) * 16) + (q & 1) * 8;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * kRow));
        vf[db] = __builtin_bit_cast(u16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    }
  }
  // scaled scores of i8 keys: (S - 128 sum q) ks, `sc` the half's 32 key scales
  VM_DEV void key_scales(f32x16& s, int u, const lds_u8* sc) {
    if constexpr (Q8) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const v4f x = *(const lds_v4f_t*)(sc + 4 * (16 * (q >> 1) + 8 * g + 4 * (q & 1)));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = BF16 ? s[4 * q + i] - qs[u] : s[4 * q + i];
          s[4 * q + i] = a * x[i];
        }
      }
    }
  }
  // -inf where the row does not see the key: past its position, before its window, or not there
  VM_DEV void mask(f32x16& s, int u, uint32_t key0, uint32_t there) {
    const int32_t hi = pos[u] - int32_t(key0), lo = D.window ? hi - int32_t(D.window) : -1;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int32_t k = 16 * (v >> 3) + 8 * int32_t(g) + (v & 7);
      if (k > hi || k <= lo || !((there >> k) & 1)) s[v] = -INFINITY;
    }
  }
  VM_DEV float top(const f32x16& s) {
    float x = s[0];
#pragma unroll
    for (int v = 1; v < 16; ++v) x = fmaxf(x, s[v]);
    return x;
  }
  // P of a half against the reference mu: two fragments, the row sums and (i8) the sums of
  // the rounded P vs
  VM_DEV void probs(const f32x16& s, float mu, const lds_u8* vs, Pf& pf0, Pf& pf1, float& rs, float& ps) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(s[8 * ks + i], sl2, -mu));
      if constexpr (Q8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) rs += e[i];
        const v4f x0 = *(const lds_v4f_t*)(vs + 4 * (16 * ks + 8 * g)), x1 = *(const lds_v4f_t*)(vs + 4 * (16 * ks + 8 * g + 4));
        // the scale of a position that is not there may be anything
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = e[i] == 0.0f ? 0.0f : e[i] * (i < 4 ? x0[i & 3] : x1[i & 3]);
      }
      const float sum = pack_p<PBF>(e, ks ? pf1 : pf0);
      if constexpr (Q8) ps += sum;
      else rs += sum;
    }
  }
  VM_DEV void rescale(int u, float a) {
    l[u] *= a;
    pv[u] *= a;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[u][db][v] *= a;
  }
  // the sums over both lanes of a row, O corrected for the i8 offset
  VM_DEV void finish(int u) {
    l[u] += xor32(l[u]);
    if constexpr (Q8) {
      const float c = 128.0f * (pv[u] + xor32(pv[u]));
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[u][db][v] -= c;
    }
  }
  // Whether O or the sum holds a NaN or an infinity (0 times either is NaN).
  VM_DEV bool not_finite(int u) const {
    float x = l[u] * 0.0f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) x = fmaf(o[u][db][v], 0.0f, x);
    return !(x == 0.0f);
  }
};

// ---- up to 64 rows ------------------------------------------------------------------------
// Per wave and stage: 32 keys of K, then of V; then, for i8, the stage's 32 key and 32
// value scales.  After the four waves' regions, a ring of table entries.
template <int HD, bool Q8>
struct PagedWaveLds {
  static constexpr uint32_t kRow = HD * (Q8 ? 1 : 2), kOp = 32 * kRow, kStage = 2 * kOp;
  static constexpr uint32_t kRegion = 32768;
  // stages that fit a wave's 32 KiB, four at most (i8 rows of 128: three, and the scales)
  static constexpr uint32_t kStages = Q8 && HD == 128 ? 3 : kRegion / kStage < 4 ? kRegion / kStage : 4;
  static constexpr uint32_t kScales = kStages * kStage;               // within the region
  static constexpr uint32_t kRounds = kOp / 1024;                      // transfers per operand
  static constexpr uint32_t kOps = 2 * kRounds + (Q8 ? 1 : 0);         // transfers per stage
  static constexpr uint32_t kRing = kWaves * kRegion;                  // [wave][stage][32] entries
  static_assert(kScales + (Q8 ? kStages * 256 : 0) <= kRegion, "a wave's stages");
  static_assert(kRing + kWaves * kStages * 128 <= 133120, "the lane's LDS");
};

// positions of each stage that are there; the waves' maxima and sums (one copy for all forms)
__shared__ uint32_t vm_paged_there[kWaves][4];
__shared__ float vm_paged_max[kWaves][64], vm_paged_sum[kWaves][64];

template <int HD, bool BF16, bool Q8, int U>
VM_LEAF bool paged_block_wave(Args A, uint32_t ti, PagedJob J) {
  A = uargs(A);
  J.uniform();
  const VM_K Task& t = task_of(A, ti);
  const PagedDesc D = paged_desc(A, t);
  typedef PagedWaveLds<HD, Q8> W;
  typedef PagedMma<HD, BF16, Q8, U> M;
  constexpr uint32_t NS = W::kStages;
  const uint32_t wave = uni(threadIdx.x >> 6);
  M B(A, t, D, J);
  B.load_rows(A, t, 0);
  const uint32_t lane = B.lane, lds0 = uint32_t(uintptr_t(B.L));
  const uint32_t mine = lds0 + wave * W::kRegion, ring = lds0 + W::kRing + wave * NS * 128;
  const lds_u8* LW = B.L + wave * W::kRegion;
  const lds_u32* LR = (const lds_u32*)(B.L + W::kRing + wave * NS * 128);
  // blocks wave, wave + 4, ... of 32 keys
  const uint32_t all = (J.k1 - J.k0 + 31) / 32, nb = all > wave ? (all - wave + 3) / 4 : 0;
  auto key0 = [&](uint32_t i) { return J.k0 + 32 * (wave + 4 * i); };
  const uint32_t l32 = lane & 31;
  const uint32_t dr = 16 * lane / W::kRow, slot = 16 * lane % W::kRow / 16;
  constexpr uint32_t kRPR = 1024 / W::kRow;                            // rows per transfer
  __syncthreads();                       // LDS free from the previous user
  auto fetch = [&](uint32_t i, int32_t page) {
    bool ok;
    const uint32_t row = B.page_row(key0(i) + l32, page, &ok), s = i % NS;
    const uint32_t there = uint32_t(__ballot(ok));
    if (lane == 0) vm_paged_there[wave][s] = there;
    const uint32_t st = mine + s * W::kStage;
#pragma unroll
    for (uint32_t j = 0; j < W::kRounds; ++j) {
      const uint32_t r = j * kRPR + dr;
      const uint64_t at = uint64_t(uint32_t(__shfl(int(row), r, 64))) * B.grow;
      dma16_at(B.kp + at + min((slot ^ pkswz<HD, Q8>(r)) * 16, B.grow - 16), uni(st + 1024 * j));
      dma16_at(B.vp + at + min((slot ^ pvswz<HD, Q8>(r)) * 16, B.grow - 16), uni(st + W::kOp + 1024 * j));
    }
    if constexpr (Q8) {
      const uint32_t rr = uint32_t(__shfl(int(row), l32, 64));
      dma4_at((const gbyte*)((lane < 32 ? B.ksc : B.vsc) + rr), uni(mine + W::kScales + s * 256));
    }
  };
  // the ring's entry of block i
  auto ahead = [&](uint32_t i) {
    if (lane < 32) dma4_at((const gbyte*)(B.table + B.entry(key0(i) + l32)), uni(ring + (i % NS) * 128));
  };
  const int32_t pos_lo = int32_t(J.pos0), pos_hi = int32_t(J.pos0 + J.tokens - 1);
  if (nb)
    for (uint32_t s = 0; s < NS; ++s) ahead(s);
  // Turn j computes block j - NS and then fills its stage with block j (the first NS turns
  // only fill): the code is laid out once, which counts where an item has few blocks (the
  // instruction cache starts cold in every launch).
  wait_vm<0>();
  for (uint32_t j = 0; j < nb + NS; ++j) {
   if (j >= NS) {
    const uint32_t i = j - NS;
    // block i has landed, and the ring's entry of block j before it: newer are the
    // transfers and entries of NS - 1 turns (fewer at the end: wait for all)
    if (j <= nb) wait_vm<(NS - 1) * (W::kOps + 1)>();
    else wait_vm<0>();
    const uint32_t s = i % NS, ka = key0(i);
    const lds_u8* K = LW + s * W::kStage;
    const lds_u8* V = K + W::kOp;
    const lds_u8* sc = LW + W::kScales + s * 256;
    const uint32_t there = uni(vm_paged_there[wave][s]);
    const bool whole = there == 0xFFFFFFFFu && int32_t(ka) + 31 <= pos_lo &&
                       (!D.window || int32_t(ka) > pos_hi - int32_t(D.window));
    if (there != 0xFFFFFFFFu && !Q8) {
      // zeros in the rows of V that hold no position of the piece
#pragma unroll
      for (uint32_t j = 0; j < W::kRounds; ++j)
        if (!((there >> (j * kRPR + dr)) & 1))
          *(lds_v4u_t*)(uintptr_t)(mine + s * W::kStage + W::kOp + 1024 * j + 16 * lane) = v4u_make(0, 0, 0, 0);
    }
    u16x8 kf[M::KS];
    f32x16 sv[U];
    typename M::Pf pf[U][2];
    B.k_frags(K, kf);
#pragma unroll
    for (int u = 0; u < U; ++u) B.scores(K, u, sv[u], kf);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      B.key_scales(sv[u], u, sc);
      if (!whole) B.mask(sv[u], u, ka, there);
      float mx = B.top(sv[u]);
      mx = fmaxf(mx, xor32(mx)) * B.sl2;
      const float mn = fmaxf(B.m[u], mx);
      if (__any(mn > B.m[u])) B.rescale(u, B.m[u] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(B.m[u] - mn));
      B.m[u] = mn;
      B.probs(sv[u], mn == -INFINITY ? 0.0f : mn, sc + 128, pf[u][0], pf[u][1], B.l[u], B.pv[u]);
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      u16x8 vf[M::DB];
      B.v_frags(V, ks, vf);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int db = 0; db < M::DB; ++db) B.o[u][db] = M::pv_mma(vf[db], pf[u][ks], B.o[u][db]);
    }
   }
   if (j < nb) {
    const int32_t page = int32_t(LR[(j % NS) * 32 + l32]);
    // this stage and ring entry have been read before they are filled
    __builtin_amdgcn_s_waitcnt(0xC07F);                                // lgkmcnt(0)
    ahead(j + NS);
    fetch(j, page);
   }
  }
  wait_vm<0>();
  // ---- join the waves -------------------------------------------------------------------
  bool bad = false;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    B.finish(u);
    if (32 * u + l32 < B.R) bad = bad || B.not_finite(u);
    if (B.g == 0) {
      vm_paged_max[wave][32 * u + l32] = B.m[u];
      vm_paged_sum[wave][32 * u + l32] = B.l[u];
    }
  }
  if (__syncthreads_or(bad)) return true;
  constexpr uint32_t DT = BF16 ? DT_BF16 : DT_F16;
  gbyte* out = resolve(A, t.dst);
  float* lf = lds_ptr<float>();
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (32u * u >= B.R) break;
    // [wave][32 rows][HD + 4] floats in the waves' own regions: rows of HD + 4 floats
    // keep the 16-byte stores of 32 lanes off each other's banks
    constexpr uint32_t LD = HD + 4;
    static_assert(32 * LD * 4 <= W::kRegion, "a wave's partial");
    float M4 = -INFINITY;
    for (uint32_t w = 0; w < uint32_t(kWaves); ++w) M4 = fmaxf(M4, vm_paged_max[w][32 * u + l32]);
    const float a = B.m[u] == -INFINITY ? 0.0f : exp2f(B.m[u] - M4);
    float* mineo = lf + wave * (W::kRegion / 4) + l32 * LD;
#pragma unroll
    for (int db = 0; db < M::DB; ++db)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *(v4f*)(mineo + 32 * db + 8 * j + 4 * B.g) = v4f_make(B.o[u][db][4 * j] * a, B.o[u][db][4 * j + 1] * a,
                                                             B.o[u][db][4 * j + 2] * a, B.o[u][db][4 * j + 3] * a);
    __syncthreads();
    // thread: four channels of a row
    const uint32_t rows = min(32u, B.R - 32 * u), per = B.hd / 4;
    for (uint32_t x = threadIdx.x; x < rows * per; x += kBlock) {
      const uint32_t r = x / per, d = x % per * 4, i = 32 * u + r;
      v4f acc = v4f_make(0, 0, 0, 0);
      float mm = -INFINITY, ls = 0.0f;
#pragma unroll
      for (uint32_t w = 0; w < uint32_t(kWaves); ++w) mm = fmaxf(mm, vm_paged_max[w][i]);
#pragma unroll
      for (uint32_t w = 0; w < uint32_t(kWaves); ++w) {
        acc += *(const v4f*)(lf + w * (W::kRegion / 4) + r * LD + d);
        const float mw = vm_paged_max[w][i];
        ls += mw == -INFINITY ? 0.0f : vm_paged_sum[w][i] * exp2f(mw - mm);
      }
      if (J.part) {
        *(v4f*)(J.part + uint64_t(i) * B.hd + d) = acc;
        if (d == 0) {
          J.part[uint64_t(B.R) * B.hd + i] = mm;
          J.part[uint64_t(B.R) * (B.hd + 1) + i] = ls;
        }
      } else {
        const uint32_t tok = B.dg.quo(i), h = J.head * B.G + i - tok * B.G;
        const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
        const float f[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
        Run<DT, 4> rn;
        rn.put(f);
        rn.store(out, (uint64_t(J.row0 + tok) * D.Hq + h) * B.hd + d);
      }
    }
    __syncthreads();
  }
  return false;
}

// Up to 16 rows, what single tokens of grouped heads have: the same on 16x16x32 products, so
// that half as many of a tile's columns are padding (with 32 the weights and the rescaling
// of rows that are not there are half of a block's instructions).  S^T of 32 keys is two
// tiles; row 4 q + i of tile k holds key 8 q + 4 k + i, so a lane's eight accumulators are
// eight consecutive keys, the second product's B operand.
template <bool BF16>
VM_DEV v4f mfma16x16(const u16x8& a, const u16x8& b, const v4f& c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
VM_DEV float quad_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
VM_DEV float quad_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

template <int HD, bool BF16, bool Q8>
VM_LEAF bool paged_block_few(Args A, uint32_t ti, PagedJob J) {
  A = uargs(A);
  J.uniform();
  const VM_K Task& t = task_of(A, ti);
  const PagedDesc D = paged_desc(A, t);
  typedef PagedWaveLds<HD, Q8> W;
  constexpr uint32_t NS = W::kStages;
  constexpr int KS = HD / 32, DT16 = HD / 16;
  constexpr bool PBF = BF16 || Q8;
  const uint32_t wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, c16 = lane & 15, l32 = lane & 31;
  const uint32_t hd = D.hd, grow = hd * (Q8 ? 1 : 2), G = D.dg.d, R = J.tokens * G;
  const gbyte* kp = resolve(A, t.b);
  const gbyte* vp = resolve(A, t.p[0]);
  const VM_G float* ksc = gcast<float>(resolve(A, t.p[1]));
  const VM_G float* vsc = gcast<float>(resolve(A, t.p[2]));
  const VM_G int32_t* table = gcast<int32_t>(resolve(A, t.p[5])) + uint64_t(J.seq) * D.MP;
  const uint32_t lds0 = uni(uint32_t(reinterpret_cast<uintptr_t>(lds_ptr<lds_u8>())));
  const uint32_t mine = lds0 + wave * W::kRegion, ring = lds0 + W::kRing + wave * NS * 128;
  const lds_u8* LW = (const lds_u8*)uintptr_t(mine);
  const lds_u32* LR = (const lds_u32*)uintptr_t(ring);
  const uint32_t all = (J.k1 - J.k0 + 31) / 32, nb = all > wave ? (all - wave + 3) / 4 : 0;
  auto key0 = [&](uint32_t i) { return J.k0 + 32 * (wave + 4 * i); };
  const uint32_t dr = 16 * lane / W::kRow, slot = 16 * lane % W::kRow / 16;
  constexpr uint32_t kRPR = 1024 / W::kRow;
  __syncthreads();                       // LDS free from the previous user
  auto ahead = [&](uint32_t i) {
    if (lane < 32) dma4_at((const gbyte*)(table + D.dp.quo(min(key0(i) + l32, J.k1 - 1))), uni(ring + (i % NS) * 128));
  };
  for (uint32_t s = 0; nb && s < NS; ++s) ahead(s);
  // q of row c16 (rows past R re-read the last), channels 32 k + 8 q ..
  const uint32_t tok = D.dg.quo(min(c16, R - 1)), row_head = J.head * G + min(c16, R - 1) - tok * G;
  const int32_t pos = int32_t(J.pos0 + tok);
  u16x8 qf[KS];
  float qs = 0.0f;
  {
    const gbyte* qb = resolve(A, t.a) + 2 * (uint64_t(J.row0 + tok) * D.ars + uint64_t(row_head) * D.ahs + D.aoff);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      qf[k] = u16x8{};
      if (32 * k + 8 * q < hd) {
        const u4 w = *(const VM_G u4*)(qb + 2 * (32 * k + 8 * q));
        qf[k] = __builtin_bit_cast(u16x8, v4u_make(w.x, w.y, w.z, w.w));
      }
      if constexpr (Q8 && BF16) qs += frag_sum<true>(qf[k]);
    }
    if constexpr (Q8 && BF16) qs = -128.0f * quad_sum(qs);
  }
  v4f o[DT16];
#pragma unroll
  for (int i = 0; i < DT16; ++i) o[i] = v4f_make(0, 0, 0, 0);
  float m = -INFINITY, l = 0.0f, pv = 0.0f;
  const float sl2 = D.scale * 1.4426950408889634f;
  const int32_t pos_lo = int32_t(J.pos0), pos_hi = int32_t(J.pos0 + J.tokens - 1);
  auto fetch = [&](uint32_t i, int32_t page) {
    const uint32_t key = key0(i) + l32, s = i % NS;
    const bool ok = key < J.k1 && page >= 0 && uint32_t(page) < D.N;
    const uint32_t row = ok ? (uint32_t(page) * D.Hkv + J.head) * D.P + (key - D.dp.quo(key) * D.P) : 0u;
    const uint32_t there = uint32_t(__ballot(ok));
    if (lane == 0) vm_paged_there[wave][s] = there;
    const uint32_t st = mine + s * W::kStage;
#pragma unroll
    for (uint32_t j = 0; j < W::kRounds; ++j) {
      const uint32_t r = j * kRPR + dr;
      const uint64_t at = uint64_t(uint32_t(__shfl(int(row), r, 64))) * grow;
      dma16_at(kp + at + min((slot ^ pkswz<HD, Q8>(r)) * 16, grow - 16), uni(st + 1024 * j));
      dma16_at(vp + at + min((slot ^ pvswz<HD, Q8>(r)) * 16, grow - 16), uni(st + W::kOp + 1024 * j));
    }
    if constexpr (Q8) dma4_at((const gbyte*)((lane < 32 ? ksc : vsc) + row), uni(mine + W::kScales + s * 256));
  };
  // turn j computes block j - NS and then fills its stage with block j, as above
  wait_vm<0>();
  for (uint32_t j = 0; j < nb + NS; ++j) {
    if (j >= NS) {
      const uint32_t i = j - NS, s = i % NS, ka = key0(i);
      if (j <= nb) wait_vm<(NS - 1) * (W::kOps + 1)>();
      else wait_vm<0>();
      const lds_u8* K = LW + s * W::kStage;
      const lds_u8* V = K + W::kOp;
      const lds_u8* sc = LW + W::kScales + s * 256;
      const uint32_t there = uni(vm_paged_there[wave][s]);
      const bool whole = there == 0xFFFFFFFFu && int32_t(ka) + 31 <= pos_lo &&
                         (!D.window || int32_t(ka) > pos_hi - int32_t(D.window));
      if (there != 0xFFFFFFFFu && !Q8) {
#pragma unroll
        for (uint32_t x = 0; x < W::kRounds; ++x)
          if (!((there >> (x * kRPR + dr)) & 1))
            *(lds_v4u_t*)(uintptr_t)(mine + s * W::kStage + W::kOp + 1024 * x + 16 * lane) = v4u_make(0, 0, 0, 0);
      }
      v4f sv[2];
      {
        u16x8 kf[2][KS];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t r = 8 * (c16 >> 2) + 4 * k + (c16 & 3), sw = pkswz<HD, Q8>(r);
#pragma unroll
          for (int x = 0; x < KS; ++x) {
            if constexpr (Q8)
              kf[k][x] = i8_frag<BF16>(*(const lds_v2u_t*)(K + r * W::kRow + (((2 * uint32_t(x) + (q >> 1)) ^ sw) * 16) + 8 * (q & 1)));
            else
              kf[k][x] = *(const lds_u16x8*)(K + r * W::kRow + (((4 * uint32_t(x) + q) ^ sw) * 16));
          }
          sv[k] = v4f_make(qs, qs, qs, qs);
        }
#pragma unroll
        for (int x = 0; x < KS; ++x)
#pragma unroll
          for (int k = 0; k < 2; ++k) sv[k] = mfma16x16<BF16>(kf[k][x], qf[x], sv[k]);
      }
      float e[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) e[x] = sv[x >> 2][x & 3];
      if constexpr (Q8) {
        const v4f x0 = *(const lds_v4f_t*)(sc + 32 * q), x1 = *(const lds_v4f_t*)(sc + 32 * q + 16);
#pragma unroll
        for (int x = 0; x < 8; ++x) e[x] *= x < 4 ? x0[x & 3] : x1[x & 3];
      }
      if (!whole) {
        const int32_t hi = pos - int32_t(ka), lo = D.window ? hi - int32_t(D.window) : -1;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int32_t k = 8 * int32_t(q) + x;
          if (k > hi || k <= lo || !((there >> k) & 1)) e[x] = -INFINITY;
        }
      }
      const float mx = quad_max(fmaxf(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])), fmaxf(fmaxf(e[4], e[5]), fmaxf(e[6], e[7])))) * sl2;
      const float mn = fmaxf(m, mx), mu = mn == -INFINITY ? 0.0f : mn;
      if (__any(mn > m)) {
        const float a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        l *= a;
        pv *= a;
#pragma unroll
        for (int x = 0; x < DT16; ++x) o[x] *= a;
        m = mn;
      }
#pragma unroll
      for (int x = 0; x < 8; ++x) e[x] = __builtin_amdgcn_exp2f(fmaf(e[x], sl2, -mu));
      if constexpr (Q8) {
        l += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
        const v4f x0 = *(const lds_v4f_t*)(sc + 128 + 32 * q), x1 = *(const lds_v4f_t*)(sc + 128 + 32 * q + 16);
#pragma unroll
        for (int x = 0; x < 8; ++x) e[x] *= x < 4 ? x0[x & 3] : x1[x & 3];
        if (!whole)                         // the scale of a position that is not there may be anything
#pragma unroll
          for (int x = 0; x < 8; ++x) e[x] = (there >> (8 * q + x)) & 1 ? e[x] : 0.0f;
      }
      PFrag<!BF16 && Q8> pf;
      const float ps = pack_p<PBF>(e, pf);
      if constexpr (Q8) pv += ps;
      else l += ps;
#pragma unroll
      for (int x = 0; x < DT16; ++x) {
        u16x8 vf;
        if constexpr (Q8) {
          const uint32_t r = 8 * q + (c16 >> 1);
          const v2i_t b = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i_t*)(V + r * W::kRow + ((uint32_t(x) ^ pvswz<HD, Q8>(r)) * 16) + 8 * (c16 & 1)));
          vf = i8_frag<true>(v2u_make(uint32_t(b.x), uint32_t(b.y)));
        } else {
          const uint32_t r = 8 * q + (c16 >> 2), z = c16 & 3;
          const lds_u8* p = V + r * W::kRow + (((2 * uint32_t(x) + (z >> 1)) ^ pvswz<HD, Q8>(r)) * 16) + (z & 1) * 8;
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * W::kRow));
          vf = __builtin_bit_cast(u16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
        o[x] = mfma16x16<PBF>(vf, pf.hi, o[x]);
        if constexpr (!BF16 && Q8) o[x] = mfma16x16<PBF>(vf, pf.lo, o[x]);
      }
    }
    if (j < nb) {
      const int32_t page = int32_t(LR[(j % NS) * 32 + l32]);
      __builtin_amdgcn_s_waitcnt(0xC07F);                                // lgkmcnt(0)
      ahead(j + NS);
      fetch(j, page);
    }
  }
  wait_vm<0>();
  // ---- join the waves -------------------------------------------------------------------
  l = quad_sum(l);
  if constexpr (Q8) {
    const float c = 128.0f * quad_sum(pv);
#pragma unroll
    for (int x = 0; x < DT16; ++x) o[x] -= c;
  }
  float z = l * 0.0f;
#pragma unroll
  for (int x = 0; x < DT16; ++x)
#pragma unroll
    for (int v = 0; v < 4; ++v) z = fmaf(o[x][v], 0.0f, z);
  if (q == 0) {
    vm_paged_max[wave][c16] = m;
    vm_paged_sum[wave][c16] = l;
  }
  if (__syncthreads_or(c16 < R && !(z == 0.0f))) return true;
  constexpr uint32_t DT = BF16 ? DT_BF16 : DT_F16;
  constexpr uint32_t LD = HD + 4;                  // floats of a row, off each other's banks
  gbyte* out = resolve(A, t.dst);
  float* lf = lds_ptr<float>();
  float M4 = -INFINITY;
  for (uint32_t w = 0; w < uint32_t(kWaves); ++w) M4 = fmaxf(M4, vm_paged_max[w][c16]);
  const float a = m == -INFINITY ? 0.0f : exp2f(m - M4);
  float* mineo = lf + wave * (W::kRegion / 4) + c16 * LD + 4 * q;
#pragma unroll
  for (int x = 0; x < DT16; ++x) *(v4f*)(mineo + 16 * x) = o[x] * a;
  __syncthreads();
  const uint32_t per = hd / 4;
  for (uint32_t x = threadIdx.x; x < R * per; x += kBlock) {
    const uint32_t i = x / per, d = x % per * 4;
    v4f acc = v4f_make(0, 0, 0, 0);
    float mm = -INFINITY, ls = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < uint32_t(kWaves); ++w) mm = fmaxf(mm, vm_paged_max[w][i]);
#pragma unroll
    for (uint32_t w = 0; w < uint32_t(kWaves); ++w) {
      acc += *(const v4f*)(lf + w * (W::kRegion / 4) + i * LD + d);
      const float mw = vm_paged_max[w][i];
      ls += mw == -INFINITY ? 0.0f : vm_paged_sum[w][i] * exp2f(mw - mm);
    }
    if (J.part) {
      *(v4f*)(J.part + uint64_t(i) * hd + d) = acc;
      if (d == 0) {
        J.part[uint64_t(R) * hd + i] = mm;
        J.part[uint64_t(R) * (hd + 1) + i] = ls;
      }
    } else {
      const uint32_t tk = D.dg.quo(i), h = J.head * G + i - tk * G;
      const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
      const float f[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
      Run<DT, 4> rn;
      rn.put(f);
      rn.store(out, (uint64_t(J.row0 + tk) * D.Hq + h) * hd + d);
    }
  }
  __syncthreads();
  return false;
}

// ---- more rows -------------------------------------------------------------------------
template <int HD, bool Q8>
struct PagedRowsLds {
  static constexpr uint32_t kRow = HD * (Q8 ? 1 : 2), kOp = 64 * kRow, kStage = 2 * kOp;
  static constexpr uint32_t kScales = 2 * kStage;                      // [stage][64 key, 64 value scales]
  static constexpr uint32_t kRounds = kOp / 4096;
  static_assert(kScales + 1024 <= 133120, "the lane's LDS");
};

template <int HD, bool BF16, bool Q8, int U>
VM_LEAF bool paged_block_rows(Args A, uint32_t ti, PagedJob J) {
  A = uargs(A);
  J.uniform();
  const VM_K Task& t = task_of(A, ti);
  const PagedDesc D = paged_desc(A, t);
  typedef PagedRowsLds<HD, Q8> W;
  typedef PagedMma<HD, BF16, Q8, U> M;
  const uint32_t wave = uni(threadIdx.x >> 6);
  M B(A, t, D, J);
  const uint32_t first = 32 * U * wave;                                // the wave's first row
  B.load_rows(A, t, first);
  const uint32_t lane = B.lane, lds0 = uint32_t(uintptr_t(B.L));
  const uint32_t nb = (J.k1 - J.k0 + 63) / 64;
  const bool wave_rows = first < B.R;
  const int32_t pos_lo = int32_t(J.pos0 + B.dg.quo(uni(min(first, B.R - 1))));
  const int32_t pos_hi = int32_t(J.pos0 + B.dg.quo(uni(min(first + 32 * U, B.R) - 1)));
  constexpr uint32_t kRPR = 4096 / W::kRow;
  const uint32_t in = 1024 * wave + 16 * lane;
  const uint32_t dr = in / W::kRow, slot = in % W::kRow / 16;
  auto fetch = [&](uint32_t kb, int32_t page, uint64_t* there) {
    bool ok;
    const uint32_t row = B.page_row(J.k0 + 64 * kb + lane, page, &ok);
    *there = __ballot(ok);
    const uint32_t st = lds0 + (kb & 1) * W::kStage + 1024 * wave;
#pragma unroll
    for (uint32_t j = 0; j < W::kRounds; ++j) {
      const uint32_t r = j * kRPR + dr;
      const uint64_t at = uint64_t(uint32_t(__shfl(int(row), r, 64))) * B.grow;
      dma16_at(B.kp + at + min((slot ^ pkswz<HD, Q8>(r)) * 16, B.grow - 16), uni(st + 4096 * j));
      dma16_at(B.vp + at + min((slot ^ pvswz<HD, Q8>(r)) * 16, B.grow - 16), uni(st + W::kOp + 4096 * j));
    }
    if constexpr (Q8) {
      if (wave < 2) dma4_at((const gbyte*)((wave == 0 ? B.ksc : B.vsc) + row), uni(lds0 + W::kScales + (kb & 1) * 512 + 256 * wave));
    }
  };
  // zeros in the rows of V that hold no position of the piece
  auto zero_rows = [&](uint32_t kb, uint64_t there) {
    if (Q8 || there == ~uint64_t(0)) return;
#pragma unroll
    for (uint32_t j = 0; j < W::kRounds; ++j)
      if (!((there >> (j * kRPR + dr)) & 1))
        *(lds_v4u_t*)(uintptr_t)(lds0 + (kb & 1) * W::kStage + W::kOp + 4096 * j + in) = v4u_make(0, 0, 0, 0);
  };
  // A masked block (and every one of a careful sweep): the online update.
  auto online = [&](int u, f32x16 (&s)[2], uint32_t ka, uint64_t there, const lds_u8* sc, typename M::Pf (&pf)[4]) {
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
      B.key_scales(s[kh], u, sc + 128 * kh);
      B.mask(s[kh], u, ka + 32 * kh, uint32_t(there >> (32 * kh)));
    }
    const float x = fmaxf(B.top(s[0]), B.top(s[1])), mn = fmaxf(B.m[u], fmaxf(x, xor32(x)) * B.sl2);
    B.rescale(u, B.m[u] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(B.m[u] - mn));
    B.m[u] = mn;
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
      B.probs(s[kh], mn == -INFINITY ? 0.0f : mn, sc + 256 + 128 * kh, pf[2 * kh], pf[2 * kh + 1], B.l[u], B.pv[u]);
  };
  // A block that every row of the wave sees whole, once every row has a reference: weights
  // against it, whatever the block's own maximum, so O is never rescaled.  A row whose
  // weights of one block sum past `bound` (P must stay finite in 16 bits) has the piece
  // swept again, carefully.
  const float bound = M::PBF ? 16777216.0f : 16384.0f;
  bool again = false;
  auto fixed = [&](int u, f32x16 (&s)[2], const lds_u8* sc, typename M::Pf (&pf)[4]) {
    float rs = 0.0f;
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
      B.key_scales(s[kh], u, sc + 128 * kh);
      B.probs(s[kh], B.m[u], sc + 256 + 128 * kh, pf[2 * kh], pf[2 * kh + 1], rs, B.pv[u]);
    }
    again = again || !(rs <= bound);
    B.l[u] += rs;
  };
  // S^T of both sub-tiles from K fragments read once, sub-tile 0's softmax while sub-tile
  // 1's S^T is on the matrix cores, then O^T of sub-tile 0 while sub-tile 1's softmax runs.
  auto body = [&](auto maskedc, const lds_u8* K, uint32_t ka, uint64_t there, const lds_u8* sc) {
    f32x16 s0[2], s1[2];
    {
      u16x8 kf[2][M::KS];
      B.k_frags(K, kf[0]);
      B.k_frags(K + 32 * W::kRow, kf[1]);
      s0[0] = s0[1] = f32x16{};
#pragma unroll
      for (int st = 0; st < M::KS; ++st)
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) s0[kh] = mfma16<BF16>(kf[kh][st], B.qf[0][st], s0[kh]);
      if constexpr (U == 2) {
        s1[0] = s1[1] = f32x16{};
#pragma unroll
        for (int st = 0; st < M::KS; ++st)
#pragma unroll
          for (int kh = 0; kh < 2; ++kh) s1[kh] = mfma16<BF16>(kf[kh][st], B.qf[1][st], s1[kh]);
      }
    }
    typename M::Pf p0[4], p1[4];
    if constexpr (decltype(maskedc)::value) online(0, s0, ka, there, sc, p0);
    else fixed(0, s0, sc, p0);
    u16x8 vf[4][M::DB];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) B.v_frags(K + W::kOp, ks, vf[ks]);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int db = 0; db < M::DB; ++db) B.o[0][db] = M::pv_mma(vf[ks][db], p0[ks], B.o[0][db]);
    if constexpr (U == 2) {
      if constexpr (decltype(maskedc)::value) online(1, s1, ka, there, sc, p1);
      else fixed(1, s1, sc, p1);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int db = 0; db < M::DB; ++db) B.o[1][db] = M::pv_mma(vf[ks][db], p1[ks], B.o[1][db]);
    }
  };
  // blocks [f0, f1) that every row of the wave sees whole
  uint32_t f0 = 0, f1 = 0;
  if (wave_rows) {
    const int32_t end = min(pos_lo, int32_t(J.k1) - 1) + 1 - int32_t(J.k0);
    f1 = end > 0 ? uint32_t(end) / 64 : 0;
    const int32_t from = D.window ? pos_hi - int32_t(D.window) + 1 - int32_t(J.k0) : 0;
    f0 = from > 0 ? (uint32_t(from) + 63) / 64 : 0;
  }
  for (uint32_t sweep = 0;; ++sweep) {
    __syncthreads();                     // LDS free from the previous user
    uint64_t there, next = 0;
    int32_t page1 = B.table[B.entry(J.k0 + 64 + lane)];
    fetch(0, B.table[B.entry(J.k0 + lane)], &there);
    wait_vm<0>();
    zero_rows(0, there);
    __syncthreads();
    auto step = [&](auto maskedc, uint32_t kb) {
      if (kb + 1 < nb) {
        fetch(kb + 1, page1, &next);
        page1 = B.table[B.entry(J.k0 + 64 * (kb + 2) + lane)];
      }
      const uint32_t ka = J.k0 + 64 * kb;
      const lds_u8* K = B.L + (kb & 1) * W::kStage;
      const lds_u8* sc = B.L + W::kScales + (kb & 1) * 512;
      if constexpr (decltype(maskedc)::value) {
        if (wave_rows && there && int32_t(ka) <= pos_hi && (!D.window || int32_t(ka) + 63 + int32_t(D.window) > pos_lo))
          body(maskedc, K, ka, there, sc);
      } else {
        again = again || there != ~uint64_t(0);         // a position without a page
        body(maskedc, K, ka, there, sc);
      }
      wait_vm<0>();
      if (kb + 1 < nb) zero_rows(kb + 1, next);
      there = next;
      __syncthreads();
    };
    // loops of their own, not one with a branch, so that each body is allocated by itself
    // (one masked loop run twice spilled: a chunk of 2048 over 8192 took 466 us, not 374);
    // block f0, the first that every row sees, gives all of them a reference
    uint32_t kb = 0;
    const uint32_t fa = sweep ? nb : min(nb, f0 + 1), fb = sweep ? nb : min(nb, f1);
    for (; kb < fa; ++kb) step(std::true_type{}, kb);
    for (; kb < fb; ++kb) step(std::false_type{}, kb);
    for (; kb < nb; ++kb) step(std::true_type{}, kb);
    if (!__syncthreads_or(again)) break;
    again = false;
    B.clear();
  }
  bool bad = false;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    B.finish(u);
    if (first + 32 * u + (lane & 31) < B.R) bad = bad || B.not_finite(u);
  }
  constexpr uint32_t DT = BF16 ? DT_BF16 : DT_F16;
  if (__syncthreads_or(bad)) return true;
  gbyte* out = resolve(A, t.dst);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t i = first + 32 * u + (lane & 31);
    if (i >= B.R) continue;
    const uint32_t tok = B.dg.quo(i), h = J.head * B.G + i - tok * B.G;
    const float inv = B.l[u] == 0.0f ? 0.0f : 1.0f / B.l[u];
#pragma unroll
    for (int db = 0; db < M::DB; ++db)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t d = 32 * db + 8 * j + 4 * B.g;
        if (d >= B.hd) continue;
        if (J.part) {
          *(v4f*)(J.part + uint64_t(i) * B.hd + d) = v4f_make(B.o[u][db][4 * j], B.o[u][db][4 * j + 1],
                                                              B.o[u][db][4 * j + 2], B.o[u][db][4 * j + 3]);
        } else {
          const float f[4] = {B.o[u][db][4 * j] * inv, B.o[u][db][4 * j + 1] * inv, B.o[u][db][4 * j + 2] * inv,
                              B.o[u][db][4 * j + 3] * inv};
          Run<DT, 4> rn;
          rn.put(f);
          rn.store(out, (uint64_t(J.row0 + tok) * D.Hq + h) * B.hd + d);
        }
      }
    if (J.part && B.g == 0) {
      J.part[uint64_t(B.R) * B.hd + i] = B.m[u];
      J.part[uint64_t(B.R) * (B.hd + 1) + i] = B.l[u];
    }
  }
  return false;
}

template <int HD, bool BF16, bool Q8>
VM_LEAF void paged_mma(Args A, uint32_t ti, uint32_t lo, uint32_t hi) {
  A = uargs(A);
  lo = uni(lo);
  hi = uni(hi);
  const VM_K Task& t = task_of(A, ti);
  const PagedDesc D = paged_desc(A, t);
  const uint32_t g = D.dg.d;
  // Rows of a block: sequences of up to 64 rows whole, longer ones in blocks of 256, or of
  // 128 where those would leave workers without one (512 tokens of 32 heads over 2048: 61 us
  // in blocks of 128, 104 of 64; of 256 114 when those of 128 took 77).
  const uint32_t r = max(uint64_t(D.T) * D.Hq >= uint64_t(t.p[7]) * 192 ? 256u : 128u, g), long_tb = r / g;
  // A key costs about 25 ns in few rows (its share of HBM) and in 128, 41 in 256; half with
  // heads of 64.
  const uint32_t unit = HD == 128 ? 2 : 1, long_weight = r > 128 ? 2 * unit : unit;
  auto tokens = [&](uint32_t n, PagedBlocks* b) {
    const bool few = n * g <= 64;
    b->weight = few ? unit : long_weight;
    b->align = r > 128 && !few ? 64 : 128;
    b->slack = few ? 640 : 1600;
    return few ? n : long_tb;
  };
  for (uint32_t w = lo; w < hi; ++w) {
    auto body = [&](const PagedJob& J) -> bool {
      const uint32_t R = J.tokens * g;
      if (R <= 16) return paged_block_few<HD, BF16, Q8>(A, ti, J);
      if (R <= 32) return paged_block_wave<HD, BF16, Q8, 1>(A, ti, J);
      if (R <= 64) return paged_block_wave<HD, BF16, Q8, 2>(A, ti, J);
      if (R <= 128) return paged_block_rows<HD, BF16, Q8, 1>(A, ti, J);
      return paged_block_rows<HD, BF16, Q8, 2>(A, ti, J);
    };
    paged_worker(A, ti, w, kMinShare, tokens, body,
                 [&](const PagedJob& J) { paged_block_generic<BF16 ? DT_BF16 : DT_F16, Q8>(A, ti, J); });
    __syncthreads();
  }
}

}  // namespace vm
