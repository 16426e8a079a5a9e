// TOP_PAGED_ATTN for f32 queries over f32 or i8 pages on the matrix cores
// (v_mfma_f32_16x16x4_f32: products and sums stay f32), heads up to 128 (multiples of 8,
// of 16 for i8), run as 64 or 128 as in tile_paged_mma.h.
//
// Blocks of up to 64 rows, 16 U of them (U = 1, 2, 4), each wave on 16-key blocks of its own
// in turn through its own LDS stages, joined at the end of the piece, as paged_block_few.
//   S^T (16 keys x 16 rows): step 4 x + i takes channel 16 x + 4 q + i in lane group q =
//   lane / 16, so a lane reads its key's channels in 16-byte runs.
//   O^T (16 channels x 16 rows) += V^T P^T: step i takes key 4 q + i, the key that the
//   lane's accumulator i of S^T holds, so P^T is those registers.
// A block of 64 rows does 16 flops a byte of LDS and is bound by the matrix cores (f32: a
// sixteenth of bf16's rate); a few rows by HBM.  Five sequences of 7 rows and 350 to 1050 keys,
// 8 / 4 heads of 96: 38 us (176 with a wave a row), most of it one item's latency.
#pragma once
#include "tile_paged_mma.h"

namespace vm {

template <int HD, bool Q8>
struct PagedF32Lds {
  static constexpr uint32_t kRow = HD * (Q8 ? 1 : 4), kOp = 16 * kRow, kStage = 2 * kOp;
  static constexpr uint32_t kRegion = 32768;
  static constexpr uint32_t kStages = kRegion / kStage < 4 ? kRegion / kStage : 4;
  static constexpr uint32_t kScales = kStages * kStage;               // i8: [stage][16 key, 16 value scales]
  static constexpr uint32_t kRounds = kOp / 1024;
  static constexpr uint32_t kOps = 2 * kRounds + (Q8 ? 1 : 0);
  static constexpr uint32_t kRing = kWaves * kRegion;                  // [wave][stage][16] entries
  static_assert(kScales + (Q8 ? kStages * 128 : 0) <= kRegion, "a wave's stages");
  static_assert(kRing + kWaves * kStages * 64 <= 133120, "the lane's LDS");
};
// Slots of the 16-byte chunks of key row r.  f32: 16 rows of K apart, V's four rows 4 q + i of a
// read in four quarters of the banks; i8: rows of K apart (V is read by bytes).
template <int HD, bool Q8>
VM_DEV uint32_t fkswz(uint32_t r) {
  if constexpr (!Q8) return r & 15;
  else return HD == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
}
template <int HD, bool Q8>
VM_DEV uint32_t fvswz(uint32_t r) {
  if constexpr (!Q8) return ((r >> 2) & 3) << 2;
  else return HD == 128 ? ((r >> 2) & 3) << 1 : (r >> 2) & 3;
}

template <int HD, bool Q8, int U>
VM_LEAF bool paged_block_f32(Args A, uint32_t ti, PagedJob J) {
  A = uargs(A);
  J.uniform();
  const VM_K Task& t = task_of(A, ti);
  const PagedDesc D = paged_desc(A, t);
  typedef PagedF32Lds<HD, Q8> W;
  constexpr uint32_t NS = W::kStages;
  constexpr int KX = HD / 16, DT16 = HD / 16;
  const uint32_t wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, c16 = lane & 15;
  const uint32_t hd = D.hd, grow = hd * (Q8 ? 1 : 4), G = D.dg.d, R = J.tokens * G;
  const gbyte* kp = resolve(A, t.b);
  const gbyte* vp = resolve(A, t.p[0]);
  const VM_G float* ksc = gcast<float>(resolve(A, t.p[1]));
  const VM_G float* vsc = gcast<float>(resolve(A, t.p[2]));
  const VM_G int32_t* table = gcast<int32_t>(resolve(A, t.p[5])) + uint64_t(J.seq) * D.MP;
  const uint32_t lds0 = uni(uint32_t(reinterpret_cast<uintptr_t>(lds_ptr<lds_u8>())));
  const uint32_t mine = lds0 + wave * W::kRegion, ring = lds0 + W::kRing + wave * NS * 64;
  const lds_u8* LW = (const lds_u8*)uintptr_t(mine);
  const lds_u32* LR = (const lds_u32*)uintptr_t(ring);
  const uint32_t all = (J.k1 - J.k0 + 15) / 16, nb = all > wave ? (all - wave + 3) / 4 : 0;
  auto key0 = [&](uint32_t i) { return J.k0 + 16 * (wave + 4 * i); };
  const uint32_t dr = 16 * lane / W::kRow, slot = 16 * lane % W::kRow / 16;
  constexpr uint32_t kRPR = W::kRow >= 1024 ? 1 : 1024 / W::kRow;
  __syncthreads();                       // LDS free from the previous user
  auto ahead = [&](uint32_t i) {
    if (lane < 16) dma4_at((const gbyte*)(table + D.dp.quo(min(key0(i) + c16, J.k1 - 1))), uni(ring + (i % NS) * 64));
  };
  for (uint32_t s = 0; nb && s < NS; ++s) ahead(s);
  float qf[U][4 * KX];
  int32_t pos[U];
  const gbyte* qb = resolve(A, t.a);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t i = min(16 * u + c16, R - 1), tok = D.dg.quo(i), h = J.head * G + i - tok * G;
    const gbyte* p = qb + 4 * (uint64_t(J.row0 + tok) * D.ars + uint64_t(h) * D.ahs + D.aoff);
    pos[u] = int32_t(J.pos0 + tok);
#pragma unroll
    for (int x = 0; x < KX; ++x) {
      u4 w = u4{0, 0, 0, 0};
      if (16 * x + 4 * q < hd) w = *(const VM_G u4*)(p + 4 * (16 * x + 4 * q));
      qf[u][4 * x] = __uint_as_float(w.x);
      qf[u][4 * x + 1] = __uint_as_float(w.y);
      qf[u][4 * x + 2] = __uint_as_float(w.z);
      qf[u][4 * x + 3] = __uint_as_float(w.w);
    }
  }
  v4f o[U][DT16];
  float m[U], l[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int i = 0; i < DT16; ++i) o[u][i] = v4f_make(0, 0, 0, 0);
    m[u] = -INFINITY;
    l[u] = 0.0f;
  }
  const float sl2 = D.scale * 1.4426950408889634f;
  const int32_t pos_lo = int32_t(J.pos0), pos_hi = int32_t(J.pos0 + J.tokens - 1);
  auto fetch = [&](uint32_t i, int32_t page) {
    const uint32_t key = key0(i) + c16, s = i % NS;
    const bool ok = key < J.k1 && page >= 0 && uint32_t(page) < D.N;
    const uint32_t row = ok ? (uint32_t(page) * D.Hkv + J.head) * D.P + (key - D.dp.quo(key) * D.P) : 0u;
    const uint32_t there = uint32_t(__ballot(ok)) & 0xFFFFu;
    if (lane == 0) vm_paged_there[wave][s] = there;
    const uint32_t st = mine + s * W::kStage;
#pragma unroll
    for (uint32_t j = 0; j < W::kRounds; ++j) {
      const uint32_t r = j * kRPR + dr;
      const uint64_t at = uint64_t(uint32_t(__shfl(int(row), r, 64))) * grow;
      dma16_at(kp + at + min((slot ^ fkswz<HD, Q8>(r)) * 16, grow - 16), uni(st + 1024 * j));
      dma16_at(vp + at + min((slot ^ fvswz<HD, Q8>(r)) * 16, grow - 16), uni(st + W::kOp + 1024 * j));
    }
    if constexpr (Q8) {
      if (lane < 32) dma4_at((const gbyte*)((lane < 16 ? ksc : vsc) + row), uni(mine + W::kScales + s * 128));
    }
  };
  // turn j computes block j - NS and then fills its stage with block j
  wait_vm<0>();
  for (uint32_t j = 0; j < nb + NS; ++j) {
    if (j >= NS) {
      const uint32_t i = j - NS, s = i % NS, ka = key0(i);
      if (j <= nb) wait_vm<(NS - 1) * (W::kOps + 1)>();
      else wait_vm<0>();
      const lds_u8* K = LW + s * W::kStage;
      const lds_u8* V = K + W::kOp;
      const lds_u8* sc = LW + W::kScales + s * 128;
      const uint32_t there = uni(vm_paged_there[wave][s]);
      const bool whole = there == 0xFFFFu && int32_t(ka) + 15 <= pos_lo &&
                         (!D.window || int32_t(ka) > pos_hi - int32_t(D.window));
      if (there != 0xFFFFu && !Q8) {
#pragma unroll
        for (uint32_t x = 0; x < W::kRounds; ++x)
          if (!((there >> (x * kRPR + dr)) & 1))
            *(lds_v4u_t*)(uintptr_t)(mine + s * W::kStage + W::kOp + 1024 * x + 16 * lane) = v4u_make(0, 0, 0, 0);
      }
      v4f sv[U];
#pragma unroll
      for (int u = 0; u < U; ++u) sv[u] = v4f_make(0, 0, 0, 0);
      const uint32_t ksw = fkswz<HD, Q8>(c16);
#pragma unroll
      for (int x = 0; x < KX; ++x) {
        float kf[4];
        if constexpr (Q8) {
          const int32_t w = *(const __attribute__((address_space(3))) int32_t*)(K + c16 * W::kRow + ((uint32_t(x) ^ ksw) * 16) + 4 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e) kf[e] = float((w << (24 - 8 * e)) >> 24);
        } else {
          const v4f w = *(const lds_v4f_t*)(K + c16 * W::kRow + (((4 * uint32_t(x) + q) ^ ksw) * 16));
#pragma unroll
          for (int e = 0; e < 4; ++e) kf[e] = w[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int u = 0; u < U; ++u) sv[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[u][4 * x + e], sv[u], 0, 0, 0);
      }
      v4f ks = v4f_make(1, 1, 1, 1), vs = v4f_make(1, 1, 1, 1);
      if constexpr (Q8) {
        ks = *(const lds_v4f_t*)(sc + 16 * q);
        vs = *(const lds_v4f_t*)(sc + 64 + 16 * q);
        if (!whole)                        // the scale of a position that is not there may be anything
#pragma unroll
          for (int e = 0; e < 4; ++e) vs[e] = (there >> (4 * q + e)) & 1 ? vs[e] : 0.0f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if constexpr (Q8) sv[u] *= ks;
        if (!whole) {
          const int32_t hi = pos[u] - int32_t(ka), lo = D.window ? hi - int32_t(D.window) : -1;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int32_t k = 4 * int32_t(q) + e;
            if (k > hi || k <= lo || !((there >> k) & 1)) sv[u][e] = -INFINITY;
          }
        }
        const float mx = quad_max(fmaxf(fmaxf(sv[u][0], sv[u][1]), fmaxf(sv[u][2], sv[u][3]))) * sl2;
        const float mn = fmaxf(m[u], mx), mu = mn == -INFINITY ? 0.0f : mn;
        if (__any(mn > m[u])) {
          const float a = m[u] == -INFINITY ? 0.0f : exp2f(m[u] - mn);
          l[u] *= a;
#pragma unroll
          for (int x = 0; x < DT16; ++x) o[u][x] *= a;
          m[u] = mn;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) sv[u][e] = exp2f(fmaf(sv[u][e], sl2, -mu));
        l[u] += (sv[u][0] + sv[u][1]) + (sv[u][2] + sv[u][3]);
        if constexpr (Q8) sv[u] *= vs;
      }
#pragma unroll
      for (int x = 0; x < DT16; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t r = 4 * q + e;
          float vf;
          if constexpr (Q8)
            vf = float(*(const __attribute__((address_space(3))) int8_t*)(V + r * W::kRow + ((uint32_t(x) ^ fvswz<HD, Q8>(r)) * 16) + c16));
          else
            vf = *(const __attribute__((address_space(3))) float*)(V + r * W::kRow + (((4 * uint32_t(x) + (c16 >> 2)) ^ fvswz<HD, Q8>(r)) * 16) + 4 * (c16 & 3));
#pragma unroll
          for (int u = 0; u < U; ++u) o[u][x] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf, sv[u][e], o[u][x], 0, 0, 0);
        }
    }
    if (j < nb) {
      const int32_t page = int32_t(LR[(j % NS) * 16 + c16]);
      __builtin_amdgcn_s_waitcnt(0xC07F);                                // lgkmcnt(0)
      ahead(j + NS);
      fetch(j, page);
    }
  }
  wait_vm<0>();
  // ---- join the waves -------------------------------------------------------------------
  float z = 0.0f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    l[u] = quad_sum(l[u]);
    if (16u * u + c16 < R) {
      z = fmaf(l[u], 0.0f, z);
#pragma unroll
      for (int x = 0; x < DT16; ++x)
#pragma unroll
        for (int v = 0; v < 4; ++v) z = fmaf(o[u][x][v], 0.0f, z);
    }
    if (q == 0) {
      vm_paged_max[wave][16 * u + c16] = m[u];
      vm_paged_sum[wave][16 * u + c16] = l[u];
    }
  }
  if (__syncthreads_or(!(z == 0.0f))) return true;
  constexpr uint32_t LD = HD + 4;                  // floats of a row, off each other's banks
  static_assert(32 * LD * 4 <= W::kRegion, "a wave's partial, two sub-tiles at a time");
  gbyte* out = resolve(A, t.dst);
  float* lf = lds_ptr<float>();
  constexpr int UB = U < 2 ? U : 2;                // sub-tiles joined at once
#pragma unroll
  for (int u0 = 0; u0 < U; u0 += UB) {
    if (16u * u0 >= R) break;
#pragma unroll
    for (int u = u0; u < u0 + UB; ++u) {
      float M4 = -INFINITY;
      for (uint32_t w = 0; w < uint32_t(kWaves); ++w) M4 = fmaxf(M4, vm_paged_max[w][16 * u + c16]);
      const float a = m[u] == -INFINITY ? 0.0f : exp2f(m[u] - M4);
      float* mineo = lf + wave * (W::kRegion / 4) + (16 * (u - u0) + c16) * LD + 4 * q;
#pragma unroll
      for (int x = 0; x < DT16; ++x) *(v4f*)(mineo + 16 * x) = o[u][x] * a;
    }
    __syncthreads();
    const uint32_t rows = min(16u * UB, R - 16 * u0), per = hd / 4;
    for (uint32_t x = threadIdx.x; x < rows * per; x += kBlock) {
      const uint32_t r = x / per, i = 16 * u0 + r, d = x % per * 4;
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
        *(v4f*)(J.part + uint64_t(i) * hd + d) = acc;
        if (d == 0) {
          J.part[uint64_t(R) * hd + i] = mm;
          J.part[uint64_t(R) * (hd + 1) + i] = ls;
        }
      } else {
        const uint32_t tk = D.dg.quo(i), h = J.head * G + i - tk * G;
        const float f[4] = {ls == 0.0f ? 0.0f : acc.x / ls, ls == 0.0f ? 0.0f : acc.y / ls,
                            ls == 0.0f ? 0.0f : acc.z / ls, ls == 0.0f ? 0.0f : acc.w / ls};
        Run<DT_F32, 4> rn;
        rn.put(f);
        rn.store(out, (uint64_t(J.row0 + tk) * D.Hq + h) * hd + d);
      }
    }
    __syncthreads();
  }
  return false;
}

template <int HD, bool Q8>
VM_LEAF void paged_f32(Args A, uint32_t ti, uint32_t lo, uint32_t hi) {
  A = uargs(A);
  lo = uni(lo);
  hi = uni(hi);
  const VM_K Task& t = task_of(A, ti);
  const PagedDesc D = paged_desc(A, t);
  const uint32_t g = D.dg.d, tb = max(1u, 64 / g);
  // a wave's 16 keys of 16 rows take about 0.9 us of matrix-core time: 64 keys and 16 rows as
  // long as streaming them from HBM (weight 4), more rows longer
  auto tokens = [&](uint32_t n, PagedBlocks* b) {
    const uint32_t rows = min(tb, n) * g;
    b->weight = rows <= 32 ? 4 : rows <= 64 ? 8 : 32;
    b->align = 64;
    b->slack = 640;
    return tb;
  };
  auto body = [&](const PagedJob& J) -> bool {
    const uint32_t R = J.tokens * g;
    if (R <= 16) return paged_block_f32<HD, Q8, 1>(A, ti, J);
    if (R <= 32) return paged_block_f32<HD, Q8, 2>(A, ti, J);
    if (R <= 64) return paged_block_f32<HD, Q8, 4>(A, ti, J);
    return true;                        // more than 64 query heads to a kv head: the general form
  };
  for (uint32_t w = lo; w < hi; ++w) {
    paged_worker(A, ti, w, g > 64 ? 2048 : 512, tokens, body, [&](const PagedJob& J) { paged_block_generic<DT_F32, Q8>(A, ti, J); });
    __syncthreads();
  }
}

VM_DEV void paged_tiles(Args A, uint32_t ti, uint32_t lo, uint32_t hi) {
  const VM_K Task& t = task_of(A, ti);
  const VM_K int32_t* d = aux_of(A) + t.p[6];
  const uint32_t dt = (t.tile_op >> 8) & 0xFF, hd = d[PD_HD];
  const bool q8 = uint32_t(d[PD_CDT]) == DT_I8;
  const bool fast = hd <= 128 && !(q8 && hd % 16);
  if (fast && dt == DT_F32) {
    if (q8) hd <= 64 ? paged_f32<64, true>(A, ti, lo, hi) : paged_f32<128, true>(A, ti, lo, hi);
    else hd <= 64 ? paged_f32<64, false>(A, ti, lo, hi) : paged_f32<128, false>(A, ti, lo, hi);
  } else if (fast && dt == DT_BF16) {
    if (q8) hd <= 64 ? paged_mma<64, true, true>(A, ti, lo, hi) : paged_mma<128, true, true>(A, ti, lo, hi);
    else hd <= 64 ? paged_mma<64, true, false>(A, ti, lo, hi) : paged_mma<128, true, false>(A, ti, lo, hi);
  } else if (fast) {
    if (q8) hd <= 64 ? paged_mma<64, false, true>(A, ti, lo, hi) : paged_mma<128, false, true>(A, ti, lo, hi);
    else hd <= 64 ? paged_mma<64, false, false>(A, ti, lo, hi) : paged_mma<128, false, false>(A, ti, lo, hi);
  } else if (q8) {
    if (dt == DT_BF16) paged_generic<DT_BF16, true>(A, ti, lo, hi);
    else if (dt == DT_F16) paged_generic<DT_F16, true>(A, ti, lo, hi);
    else paged_generic<DT_F32, true>(A, ti, lo, hi);
  } else {
    if (dt == DT_BF16) paged_generic<DT_BF16, false>(A, ti, lo, hi);
    else if (dt == DT_F16) paged_generic<DT_F16, false>(A, ti, lo, hi);
    else paged_generic<DT_F32, false>(A, ti, lo, hi);
  }
}

}  // namespace vm
