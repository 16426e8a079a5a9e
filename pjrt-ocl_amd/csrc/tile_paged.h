// TOP_PAGED_ATTN (extension): causal attention of a step's rows over the pages of a
// cache, chunks of new tokens and single tokens in one batch.
//
//   out[r, h] = sum_j softmax_j(scale q[r, h] . k_j) v_j
//
// over the positions j of row r's sequence with j <= p and, with a window, j > p - window,
// p the row's own position (tile_cache.h describes a step's rows and the pages).  Query
// head h reads kv head h / g, g = Hq / Hkv.  Positions whose table entry is no page are
// not seen; rows that see nothing are 0, as are rows of no sequence and rows of a
// sequence whose length is less than its new rows or more than its pages hold.
//
// Work.  The lengths are known on the device only, so the task has a fixed number of
// workers (p7, one per lane) that divide the step among themselves.  A sequence's new
// tokens are cut into blocks of TB tokens; an item is one block of one kv head, its rows
// all (token, query head of the group) pairs, its keys [kstart, kend) from the first
// position its first token sees to its last token's own.  An item costs kItemCost +
// its keys; with C the sum over all items, in the order sequence, head, block, worker w
// takes cost [w C / W, (w + 1) C / W).  An item that lies across workers is cut at
// multiples of kKeyAlign keys: each piece leaves its rows' (max, sum, O) in the task's
// scratch, and the piece that arrives last at the item's counter joins them in key
// order.  So one long sequence and many short ones keep every CU as busy, the result
// depends on the lengths alone, and nothing waits.
//
// Scratch: 2 W slots of kPagedMaxRows' (or T g) rows x (hd + 2) floats: worker w's first
// item in slot 2 w, its last in 2 w + 1; then W arrival counters, by the worker that
// holds the item's first cost.
#pragma once
#include "tile_attn.h"
#include "tile_cache.h"

namespace vm {

constexpr uint32_t kItemCost = 96;         // an item's fixed cost in keys
constexpr uint32_t kKeyAlign = 128;        // pieces of an item are multiples of this many keys
constexpr uint32_t kMinShare = 256;        // cost of a worker at least (> kItemCost + kKeyAlign: see pieces())

struct PagedSeq {                          // a sequence with new rows and a place for them
  uint32_t r0, n, len, p0;                 // first row, rows, length, first row's position
};
// Sequence s, false when it has no rows or its length does not fit them; `bad`: it has
// rows that must be 0.
VM_DEV bool paged_seq(const PagedDesc& D, int32_t c0, int32_t c1, int32_t len, PagedSeq* q, bool* bad) {
  const uint32_t a = uint32_t(min(max(c0, 0), int32_t(D.T))), b = uint32_t(min(max(c1, 0), int32_t(D.T)));
  q->r0 = a;
  q->n = b > a ? b - a : 0;
  q->len = uint32_t(len);
  q->p0 = uint32_t(len) - q->n;
  *bad = q->n && (len < int32_t(q->n) || uint32_t(len) > D.MP * D.P);
  return q->n && !*bad;
}

// Blocks of a sequence: key ranges and the cost of the first b blocks of a head.
struct PagedBlocks {
  uint32_t tb, nb, n, p0, len, window;
  VM_DEV uint32_t kend(uint32_t b) const { return p0 + min(n, (b + 1) * tb); }
  VM_DEV uint32_t kstart(uint32_t b) const {
    if (!window) return 0;
    const int64_t k = int64_t(p0) + int64_t(b) * tb + 1 - window;
    return k > 0 ? uint32_t(k) : 0u;
  }
  // sum over i < b of kItemCost + kend(i) - kstart(i)
  VM_DEV uint64_t before(uint32_t b) const {
    uint64_t c = uint64_t(b) * (kItemCost + p0) + uint64_t(tb) * (uint64_t(b) * (b + 1) / 2);
    if (b == nb) c -= uint64_t(nb) * tb - n;                       // the last block's end is the length
    if (window) {
      const int64_t a = int64_t(p0) + 1 - window;                  // kstart(i) = max(0, a + i tb)
      const uint64_t i0 = a > 0 ? 0 : uint64_t(-a) / tb + 1;       // the first i with a + i tb > 0
      if (b > i0) {
        const uint64_t cnt = b - i0;
        c -= cnt * uint64_t(a + int64_t(i0 * tb)) + uint64_t(tb) * (cnt * (cnt - 1) / 2);
      }
    }
    return c;
  }
};

// One piece of an item.
struct PagedJob {
  uint32_t seq, head, row0, tokens, pos0;  // rows row0 .. + tokens - 1 of the step, at positions pos0 ..
  uint32_t k0, k1;                         // its keys
  float* part;                             // its partial slot (null: the whole item, written to the output)
};

VM_DEV void agent_store(float* p, float v) {
  __hip_atomic_store(reinterpret_cast<uint32_t*>(p), __float_as_uint(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
VM_DEV float agent_load(const float* p) {
  return __uint_as_float(
      __hip_atomic_load(reinterpret_cast<const uint32_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Partial slot of R rows: O [R][hd], then maxima [R] (base 2, scaled) and sums [R].
VM_DEV uint64_t paged_slot_floats(const PagedDesc& D) {
  const uint64_t rows = uint64_t(D.T) * (D.Hq / D.Hkv);
  return (rows < kPagedMaxRows ? rows : kPagedMaxRows) * (D.hd + 2);
}

// Zeros in the rows that no valid sequence has, a share per worker.
VM_DEV void paged_zero_rows(Args A, const VM_K Task& t, const PagedDesc& D, uint32_t w, const VM_G int32_t* cu,
                            const VM_G int32_t* lens, bool any_bad) {
  const uint32_t dt = (t.tile_op >> 8) & 0xFF, W = t.p[7];
  gbyte* out = resolve(A, t.dst);
  const uint32_t per = D.Hq * D.hd;
  auto zero = [&](uint32_t a, uint32_t b) {
    for (uint32_t r = a + w; r < b; r += W)
      for (uint32_t i = threadIdx.x; i < per; i += kBlock) store_f(out, dt, uint64_t(r) * per + i, 0.0f);
  };
  const int32_t first = cu[0], last = cu[D.B];
  zero(0, uint32_t(min(max(first, 0), int32_t(D.T))));
  zero(uint32_t(min(max(last, 0), int32_t(D.T))), D.T);
  for (uint32_t s = 0; any_bad && s < D.B; ++s) {
    PagedSeq q;
    bool bad;
    paged_seq(D, cu[s], cu[s + 1], lens[s], &q, &bad);
    if (bad) zero(q.r0, q.r0 + q.n);
  }
}

// Join the pieces of an item: R rows, np partials, piece i in slot(i).  Every thread of
// the block calls it, after the last arrival.
template <class Slot, class Row>
VM_DEV void paged_join(Args A, const VM_K Task& t, const PagedDesc& D, uint32_t R, uint32_t np, Slot slot, Row row_at) {
  const uint32_t dt = (t.tile_op >> 8) & 0xFF, hd = D.hd;
  gbyte* out = resolve(A, t.dst);
  // a thread owns channels d, d + cols, ... of rows r, r + rpp, ...
  const uint32_t cols = min(256u, pow2_at_least(hd)), rpp = kBlock / cols;
  const uint32_t d0 = threadIdx.x % cols;
  for (uint32_t r = threadIdx.x / cols; r < R; r += rpp) {
    float M = -INFINITY;
    for (uint32_t i = 0; i < np; ++i) M = fmaxf(M, agent_load(slot(i) + uint64_t(R) * hd + r));
    float L = 0.0f, O = 0.0f;
    for (uint32_t i = 0; i < np; ++i) {
      const float* p = slot(i);
      const float m = agent_load(p + uint64_t(R) * hd + r), l = agent_load(p + uint64_t(R) * (hd + 1) + r);
      const float o = d0 < hd ? agent_load(p + uint64_t(r) * hd + d0) : 0.0f;
      const float a = m == -INFINITY ? 0.0f : exp2f(m - M);
      L = fmaf(l, a, L);
      O = fmaf(o, a, O);
    }
    if (d0 < hd) store_f(out, dt, row_at(r) + d0, L == 0.0f ? 0.0f : O / L);
  }
}

// Worker w's share: its items' pieces one after another.  tokens_per_block(n) -> TB;
// body(job) computes a piece (every thread of the block).
template <class Tokens, class Body>
VM_DEV void paged_worker(Args A, uint32_t ti, uint32_t w, Tokens tokens_per_block, Body body) {
  const VM_K Task& t = task_of(A, ti);
  const PagedDesc D = paged_desc(A, t);
  const uint32_t W = t.p[7], tid = threadIdx.x, g = D.Hq / D.Hkv;
  const VM_G int32_t* cu = gcast<int32_t>(resolve(A, t.p[3]));
  const VM_G int32_t* lens = gcast<int32_t>(resolve(A, t.p[4]));
  __shared__ uint64_t s_wave[kWaves + 2];
  __shared__ uint32_t s_last;

  auto blocks = [&](const PagedSeq& q) {
    PagedBlocks b;
    b.tb = tokens_per_block(q.n);
    b.nb = (q.n + b.tb - 1) / b.tb;
    b.n = q.n;
    b.p0 = q.p0;
    b.len = q.len;
    b.window = D.window;
    return b;
  };
  // cost of the thread's sequences, and its sum before them
  const uint32_t per = (D.B + kBlock - 1) / kBlock, first = min(D.B, tid * per), last = min(D.B, first + per);
  uint64_t own = 0;
  bool any_bad = false, outside = false;
  for (uint32_t s = first; s < last; ++s) {
    PagedSeq q;
    bool bad;
    const int32_t c0 = cu[s], c1 = cu[s + 1];
    if (paged_seq(D, c0, c1, lens[s], &q, &bad)) {
      const PagedBlocks b = blocks(q);
      own += D.Hkv * b.before(b.nb);
    }
    any_bad = any_bad || bad;
    outside = outside || (s == 0 && c0 > 0) || (s == D.B - 1 && c1 < int32_t(D.T));
  }
  uint64_t sum = own;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    const uint64_t o = __shfl_up(sum, k, 64);
    if ((tid & 63) >= uint32_t(k)) sum += o;
  }
  __syncthreads();
  if ((tid & 63) == 63) s_wave[tid >> 6] = sum;
  any_bad = __syncthreads_or(any_bad);
  outside = __syncthreads_or(outside);
  uint64_t before = sum - own, total = 0;
#pragma unroll
  for (uint32_t k = 0; k < uint32_t(kWaves); ++k) {
    if (k < (tid >> 6)) before += s_wave[k];
    total += s_wave[k];
  }
  if (any_bad || outside) paged_zero_rows(A, t, D, w, cu, lens, any_bad);
  const uint64_t share = max(uint64_t(kMinShare), (total + W - 1) / W);
  const uint64_t c0 = w * share, c1 = min(total, c0 + share);
  if (c0 >= total) return;
  // the sequence of cost c0
  if (own && before <= c0 && c0 < before + own) {
    uint64_t base = before;
    for (uint32_t s = first; s < last; ++s) {
      PagedSeq q;
      bool bad;
      if (!paged_seq(D, cu[s], cu[s + 1], lens[s], &q, &bad)) continue;
      const PagedBlocks b = blocks(q);
      const uint64_t c = D.Hkv * b.before(b.nb);
      if (c0 < base + c) {
        s_wave[kWaves] = base;
        s_wave[kWaves + 1] = s;
        break;
      }
      base += c;
    }
  }
  __syncthreads();
  auto uni64 = [](uint64_t x) { return (uint64_t(uni(uint32_t(x >> 32))) << 32) | uni(uint32_t(x)); };
  uint64_t base = uni64(s_wave[kWaves]);
  uint32_t s = uni(uint32_t(s_wave[kWaves + 1]));

  float* scratch = reinterpret_cast<float*>(A->scratch + A->task_scratch[ti]);
  const uint64_t slot_floats = paged_slot_floats(D);
  uint32_t* arrivals = reinterpret_cast<uint32_t*>(scratch + 2 * uint64_t(W) * slot_floats);

  for (; s < D.B && base < c1; ++s) {
    PagedSeq q;
    bool bad;
    if (!paged_seq(D, uni(cu[s]), uni(cu[s + 1]), uni(lens[s]), &q, &bad)) continue;
    const PagedBlocks B = blocks(q);
    const uint64_t S1 = B.before(B.nb);                        // a head's cost
    uint32_t h = 0, b = 0;
    if (c0 > base) {
      const uint64_t x = c0 - base;
      h = uint32_t(x / S1);
      const uint64_t rem = x - h * S1;
      uint32_t lo = 0, hi = B.nb;                              // the last b with before(b) <= rem
      while (hi - lo > 1) {
        const uint32_t m = (lo + hi) / 2;
        if (B.before(m) <= rem) lo = m;
        else hi = m;
      }
      b = lo;
    }
    for (; h < D.Hkv; ++h, b = 0) {
      bool done = false;
      for (; b < B.nb; ++b) {
        const uint64_t I0 = base + h * S1 + B.before(b);
        if (I0 >= c1) {
          done = true;
          break;
        }
        const uint32_t ks = B.kstart(b), K = B.kend(b) - ks;
        const uint64_t I1 = I0 + kItemCost + K;
        // Keys of the item before worker boundary c: a multiple of kKeyAlign.  The first
        // piece can be empty (the boundary lies in the item's fixed cost or within
        // kKeyAlign keys of its start); no other can, since a share is more than kItemCost +
        // kKeyAlign and the last boundary lies before the item's end.
        auto keys_before = [&](uint64_t c) -> uint32_t {
          if (c <= I0 + kItemCost) return 0;
          if (c >= I1) return K;
          return uint32_t(c - I0 - kItemCost) / kKeyAlign * kKeyAlign;
        };
        const uint32_t ka = I0 >= c0 ? 0 : keys_before(c0), kb = I1 <= c1 ? K : keys_before(c1);
        if (ka >= kb) continue;
        const uint32_t tok0 = b * B.tb;
        PagedJob job;
        job.seq = s;
        job.head = h;
        job.row0 = q.r0 + tok0;
        job.tokens = min(B.tb, q.n - tok0);
        job.pos0 = q.p0 + tok0;
        job.k0 = ks + ka;
        job.k1 = ks + kb;
        job.part = nullptr;
        if (ka == 0 && kb == K) {
          body(job);
          continue;
        }
        const uint32_t w0 = uint32_t(I0 / share), w1 = uint32_t((I1 - 1) / share);
        const uint32_t skip = keys_before((w0 + 1) * share) == 0 ? 1u : 0u;
        const uint32_t np = w1 - w0 + 1 - skip;
        job.part = scratch + (w == w0 ? 2 * uint64_t(w) + 1 : 2 * uint64_t(w)) * slot_floats;
        body(job);
        // the barrier orders every thread's stores (done: vmcnt 0) before thread 0's
        // arrival, an agent-scope acquire-release; the last one sees every piece
        __builtin_amdgcn_s_waitcnt(0x0F70);
        __syncthreads();
        if (tid == 0) {
          const uint32_t n = __hip_atomic_fetch_add(arrivals + w0, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
          if (n == np - 1) __hip_atomic_store(arrivals + w0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          s_last = n == np - 1;
        }
        __syncthreads();
        if (s_last) {
          const uint32_t R = job.tokens * g;
          auto slot = [&](uint32_t i) -> const float* {
            const uint32_t v = w0 + skip + i;
            return scratch + (v == w0 ? 2 * uint64_t(v) + 1 : 2 * uint64_t(v)) * slot_floats;
          };
          auto row_at = [&](uint32_t r) -> uint64_t {
            return (uint64_t(job.row0 + r / g) * D.Hq + h * g + r % g) * D.hd;
          };
          paged_join(A, t, D, R, np, slot, row_at);
        }
        __syncthreads();
      }
      if (done) break;
    }
    base += D.Hkv * S1;
  }
}

// ---- any type and head size ---------------------------------------------------------------
// One wave per row: a lane scores its key of a 64-key chunk (its own row of K, in 8-element
// runs, against q in LDS), then lane groups of hd / 8 add the chunk's values, 8 channels a
// lane.  Invisible positions are left out of both sums, whatever their pages hold.
// Sums f32, one rounding at the output.
constexpr uint32_t kPagedGenericRows = 32;

template <uint32_t DT, bool Q8>
VM_DEV void paged_block_generic(Args A, const VM_K Task& t, const PagedDesc& D, const PagedJob& J) {
  const uint32_t lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), g = D.Hq / D.Hkv, hd = D.hd;
  const gbyte* qb = resolve(A, t.a);
  const gbyte* kp = resolve(A, t.b);
  const gbyte* vp = resolve(A, t.p[0]);
  const VM_G float* ksc = gcast<float>(resolve(A, t.p[1]));
  const VM_G float* vsc = gcast<float>(resolve(A, t.p[2]));
  const VM_G int32_t* table = gcast<int32_t>(resolve(A, t.p[5])) + uint64_t(J.seq) * D.MP;
  gbyte* out = resolve(A, t.dst);
  typedef __attribute__((address_space(3))) float lds_f;
  lds_f* ql = (lds_f*)lds_ptr<float>() + wave * kPagedMaxHd;
  const uint32_t lph = pow2_at_least(hd / 8), l = lane & (lph - 1), grp = lane / lph, ngrp = 64 / lph;
  const uint32_t c = min(l, hd / 8 - 1) * 8;
  const float sl2 = D.scale * 1.4426950408889634f;
  const uint32_t R = J.tokens * g;
  typedef Run<DT, 8> Rn;
  auto load8 = [&](const gbyte* base, uint64_t e, float (&f)[8]) {
    if constexpr (Q8) {
      i8_get(*(const VM_G v2u*)(base + e), f);
    } else {
      Rn r;
      r.load(base, e);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = r.get(i);
    }
  };
  __syncthreads();
  for (uint32_t i = wave; i < R; i += kWaves) {
    const uint32_t tok = i / g, hq = J.head * g + i % g, p = J.pos0 + tok;
    const uint64_t qe = uint64_t(J.row0 + tok) * D.ars + uint64_t(hq) * D.ahs + D.aoff;
    for (uint32_t d = lane; d < hd; d += 64) ql[d] = load_f(qb, DT, qe + d);
    __builtin_amdgcn_wave_barrier();
    // the row's keys within the piece
    const uint32_t lo = D.window && p + 1 > D.window ? max(J.k0, p + 1 - D.window) : J.k0, hi = min(J.k1, p + 1);
    float m = -INFINITY, lsum = 0.0f, o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = 0.0f;
    for (uint32_t kb = lo; kb < hi; kb += 64) {
      const uint32_t key = kb + lane;
      const uint32_t kk = min(key, hi - 1), pi = kk / D.P;
      const int32_t page = table[pi];
      const bool see = key < hi && page >= 0 && uint32_t(page) < D.N;
      const uint64_t row = see ? (uint64_t(page) * D.Hkv + J.head) * D.P + (kk - pi * D.P) : 0;
      float acc = 0.0f;
      for (uint32_t d = 0; d < hd; d += 8) {
        float f[8];
        load8(kp, row * hd + d, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc = fmaf(ql[d + j], f[j], acc);
      }
      if constexpr (Q8) acc *= ksc[row];
      const float sc = see ? acc * sl2 : -INFINITY;
      const float mn = fmaxf(m, wave_max(sc)), mu = mn == -INFINITY ? 0.0f : mn;
      const float al = m == -INFINITY ? 0.0f : exp2f(m - mu);
      float pr = see ? exp2f(sc - mu) : 0.0f;
      lsum = lsum * al + wave_sum(pr);
      m = mn;
      if constexpr (Q8) pr *= see ? vsc[row] : 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] *= al;
      const uint32_t cnt = min(64u, hi - kb);
      for (uint32_t j0 = 0; j0 < cnt; j0 += ngrp) {
        const uint32_t j = min(j0 + grp, 63u);
        const float pj = __shfl(pr, j, 64);
        const uint32_t rl = __shfl(uint32_t(row), j, 64), rh = __shfl(uint32_t(row >> 32), j, 64);
        const bool sj = __shfl(int(see), j, 64) && j0 + grp < cnt;
        float f[8];
        load8(vp, ((uint64_t(rh) << 32) | rl) * hd + c, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = sj ? fmaf(pj, f[e], o[e]) : o[e];
      }
    }
    for (uint32_t msk = lph; msk < 64; msk <<= 1)
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] += __shfl_xor(o[e], msk, 64);
    if (J.part) {
      if (lane < hd / 8)
#pragma unroll
        for (int e = 0; e < 8; ++e) agent_store(J.part + uint64_t(i) * hd + c + e, o[e]);
      if (lane == 0) {
        agent_store(J.part + uint64_t(R) * hd + i, m);
        agent_store(J.part + uint64_t(R) * (hd + 1) + i, lsum);
      }
    } else if (lane < hd / 8) {
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = lsum == 0.0f ? 0.0f : o[e] / lsum;
      Rn r;
      r.put(o);
      r.store(out, (uint64_t(J.row0 + tok) * D.Hq + hq) * hd + c);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <uint32_t DT, bool Q8>
VM_TILE void paged_generic(Args A, uint32_t ti, uint32_t lo, uint32_t hi) {
  A = uargs(A);
  lo = uni(lo);
  hi = uni(hi);
  const VM_K Task& t = task_of(A, ti);
  const PagedDesc D = paged_desc(A, t);
  const uint32_t g = D.Hq / D.Hkv;
  for (uint32_t w = lo; w < hi; ++w) {
    paged_worker(A, ti, w, [&](uint32_t) { return max(1u, kPagedGenericRows / g); },
                 [&](const PagedJob& J) { paged_block_generic<DT, Q8>(A, t, D, J); });
    __syncthreads();
  }
}

VM_DEV void paged_tiles(Args A, uint32_t ti, uint32_t lo, uint32_t hi) {
  const VM_K Task& t = task_of(A, ti);
  const uint32_t dt = (t.tile_op >> 8) & 0xFF;
  const bool q8 = uint32_t((aux_of(A) + t.p[6])[PD_CDT]) == DT_I8;
  if (q8) {
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
