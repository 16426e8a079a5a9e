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
// position its first token sees to its last token's own.  An item costs kItemCost plus
// its keys times the block's weight (what a key costs a block of its rows); with C the
// sum over all items, in the order sequence, head, block, worker w takes cost
// [w C / W, (w + 1) C / W).  An item that lies across workers is cut, unless that is near
// its start or end: each piece leaves its rows' (max, sum, O) in the task's
// scratch, and the piece that arrives last at the item's counter joins them in key
// order.  So one long sequence and many short ones keep every CU as busy, the result
// depends on the lengths alone, and nothing waits.
//
// Scratch: kMaxLanes arrival counters, by the worker of the item's first piece, 0 between
// tasks (tasks that share the scratch have partials of other sizes, so the counters come
// first); then 2 W slots of kPagedMaxRows' (or T g) rows x (hd + 2) floats: worker w's piece
// of an item that begins before it in slot 2 w, of one that ends after it in 2 w + 1.
#pragma once
#include "tile_attn.h"
#include "tile_cache.h"

namespace vm {

// Costs are in units of about 12.5 ns of one CU: what a key of 128 channels costs a block of
// 64 rows on the matrix cores, half of what streaming it from HBM costs (all CUs at once).
constexpr uint32_t kItemCost = 448;        // an item's fixed cost
constexpr uint32_t kMinShare = 512;        // cost of a worker at least

struct PagedSeq {                          // a sequence with new rows and a place for them
  uint32_t r0, n, len, p0;                 // first row, rows, length, first row's position
};
// Sequence s, false when it has no rows of the step, some of its rows are not the step's or its
// length does not fit them; `bad`: it has rows that must be 0.
VM_DEV bool paged_seq(const PagedDesc& D, int32_t c0, int32_t c1, int32_t len, PagedSeq* q, bool* bad) {
  const uint32_t a = uint32_t(min(max(c0, 0), int32_t(D.T))), b = uint32_t(min(max(c1, 0), int32_t(D.T)));
  q->r0 = a;
  q->n = b > a ? b - a : 0;
  q->len = uint32_t(len);
  q->p0 = uint32_t(len) - q->n;
  *bad = q->n && (c0 < 0 || c1 > int32_t(D.T) || len < int32_t(q->n) || uint32_t(len) > D.MP * D.P);
  return q->n && !*bad;
}

// Blocks of a sequence: key ranges and the cost of the first b blocks of a head.
struct PagedBlocks {
  uint32_t tb, nb, n, p0, weight, align;   // cut at multiples of `align` keys; weight a power of two
  uint32_t slack;                          // cost that a piece is worth at least
  int32_t a;                     // kstart(b) = max(0, a + b tb)
  uint32_t i0;                   // the first b with a + b tb > 0
  VM_DEV void set(const PagedSeq& q, uint32_t window) {
    nb = q.n <= tb ? 1u : (q.n + tb - 1) / tb;
    n = q.n;
    p0 = q.p0;
    a = INT32_MIN;
    i0 = 0xFFFFFFFFu;
    if (window) {
      a = int32_t(p0) + 1 - int32_t(window);
      i0 = a > 0 ? 0u : uint32_t(-a) / tb + 1;
    }
  }
  VM_DEV uint32_t kend(uint32_t b) const { return p0 + min(n, (b + 1) * tb); }
  VM_DEV uint32_t kstart(uint32_t b) const { return b < i0 ? 0u : uint32_t(a + int32_t(b * tb)); }
  // sum over i < b of kItemCost + weight (kend(i) - kstart(i))
  VM_DEV uint64_t before(uint32_t b) const {
    uint64_t c = uint64_t(b) * p0 + uint64_t(tb) * (uint64_t(b) * (b + 1) / 2);
    if (b == nb) c -= nb * tb - n;                               // the last block's end is the length
    if (b > i0) {
      const uint64_t cnt = b - i0;
      c -= cnt * uint32_t(a + int32_t(i0 * tb)) + uint64_t(tb) * (cnt * (cnt - 1) / 2);
    }
    return c * weight + uint64_t(b) * kItemCost;
  }
};

// One piece of an item.
struct PagedJob {
  uint32_t seq, head, row0, tokens, pos0;  // rows row0 .. + tokens - 1 of the step, at positions pos0 ..
  uint32_t k0, k1;                         // its keys
  float* part;                             // its partial slot (null: the whole item, written to the output)
  // a job passed to a function arrives in vector registers
  VM_DEV void uniform() {
    seq = uni(seq);
    head = uni(head);
    row0 = uni(row0);
    tokens = uni(tokens);
    pos0 = uni(pos0);
    k0 = uni(k0);
    k1 = uni(k1);
    part = uni_ptr(part);
  }
};

// Partial slot of R rows: O [R][hd], then maxima [R] (base 2, scaled) and sums [R].
VM_DEV uint64_t paged_slot_floats(const PagedDesc& D) {
  const uint64_t rows = uint64_t(D.T) * (D.Hq / D.Hkv);
  return ((rows < kPagedMaxRows ? rows : kPagedMaxRows) * (D.hd + 2) + 3) & ~uint64_t(3);   // whole 16 bytes
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
// the block calls it, after the last arrival.  Each row's weights first (a thread a row,
// into LDS), then a thread takes four channels of a row; the pieces' loads are issued
// eight at a time (one after another they cost a memory round trip each: a 256-row item
// of three pieces took 60 us to join, with them together 8).
template <class Slot, class Row>
VM_DEV void paged_join(Args A, const VM_K Task& t, const PagedDesc& D, uint32_t R, uint32_t np, Slot slot, Row row_at) {
  const uint32_t dt = (t.tile_op >> 8) & 0xFF, hd = D.hd, per = hd / 4, tid = threadIdx.x;
  gbyte* out = resolve(A, t.dst);
  float* wt = lds_ptr<float>();                          // [np][rows of the round]
  const uint32_t rc = min(R, 32768u / np);               // np <= 4096 workers
  constexpr uint32_t U = 8;
  for (uint32_t r0 = 0; r0 < R; r0 += rc) {
    const uint32_t rows = min(rc, R - r0);
    __syncthreads();
    for (uint32_t r = tid; r < rows; r += kBlock) {
      const uint64_t at = uint64_t(R) * hd + r0 + r;
      float M = -INFINITY, L = 0.0f;
      for (uint32_t i0 = 0; i0 < np; i0 += U) {
        float m[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) m[u] = slot(min(i0 + u, np - 1))[at];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
          M = fmaxf(M, m[u]);
          if (i0 + u < np) wt[(i0 + u) * rows + r] = m[u];
        }
      }
      for (uint32_t i0 = 0; i0 < np; i0 += U) {
        float l[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) l[u] = slot(min(i0 + u, np - 1))[at + R];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
          if (i0 + u < np) {
            float* w = wt + (i0 + u) * rows + r;
            const float a = *w == -INFINITY ? 0.0f : exp2f(*w - M);
            L = fmaf(l[u], a, L);
            *w = a;
          }
      }
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;     // a row that saw nothing is 0
      for (uint32_t i = 0; i < np; ++i) wt[i * rows + r] *= inv;
    }
    __syncthreads();
    for (uint32_t x = tid; x < rows * per; x += kBlock) {
      const uint32_t r = x / per, d = x % per * 4;
      v4f O = v4f_make(0, 0, 0, 0);
      for (uint32_t i0 = 0; i0 < np; i0 += U) {
        v4f o[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) o[u] = *(const v4f*)(slot(min(i0 + u, np - 1)) + uint64_t(r0 + r) * hd + d);
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
          const float a = i0 + u < np ? wt[(i0 + u) * rows + r] : 0.0f;
          if (i0 + u < np)
#pragma unroll
            for (int e = 0; e < 4; ++e) O[e] = fmaf(o[u][e], a, O[e]);
        }
      }
      const uint64_t at = row_at(r0 + r) + d;
      const float f[4] = {O[0], O[1], O[2], O[3]};
      if (dt == DT_F32) {
        Run<DT_F32, 4> q;
        q.put(f);
        q.store(out, at);
      } else if (dt == DT_BF16) {
        Run<DT_BF16, 4> q;
        q.put(f);
        q.store(out, at);
      } else {
        Run<DT_F16, 4> q;
        q.put(f);
        q.store(out, at);
      }
    }
  }
}

__shared__ uint64_t vm_paged_cost[kWaves + 2];   // waves' sums, then the first sequence and the cost before it
__shared__ uint32_t vm_paged_last;
// the step's first kPagedHeld sequences: first row, end row, length
constexpr uint32_t kPagedHeld = 256;
__shared__ int32_t vm_paged_seq[3][kPagedHeld];

// Worker w's share: its items' pieces one after another.  tokens_per_block(n, &blocks) -> TB
// sets weight, align and slack; align * weight is at most `min_share`; body(job) computes a
// piece (every thread of the block) and says whether redo(job) has to.
template <class Tokens, class Body, class Redo>
VM_DEV void paged_worker(Args A, uint32_t ti, uint32_t w, uint32_t min_share, Tokens tokens_per_block, Body body,
                         Redo redo) {
  const VM_K Task& t = task_of(A, ti);
  const PagedDesc D = paged_desc(A, t);
  const uint32_t W = t.p[7], tid = threadIdx.x, g = D.Hq / D.Hkv;
  const VM_G int32_t* cu = gcast<int32_t>(resolve(A, t.p[3]));
  const VM_G int32_t* lens = gcast<int32_t>(resolve(A, t.p[4]));
  auto blocks = [&](const PagedSeq& q) {
    PagedBlocks b;
    b.tb = tokens_per_block(q.n, &b);
    b.set(q, D.window);
    return b;
  };
  auto sequence = [&](uint32_t s, PagedSeq* q) {
    bool bad;
    return s < kPagedHeld ? paged_seq(D, uni(vm_paged_seq[0][s]), uni(vm_paged_seq[1][s]), uni(vm_paged_seq[2][s]), q, &bad)
                          : paged_seq(D, uni(cu[s]), uni(cu[s + 1]), uni(lens[s]), q, &bad);
  };
  __syncthreads();                          // a worker before this one has read what it held
  // cost of the thread's sequences, and its sum before them
  const uint32_t per = (D.B + kBlock - 1) / kBlock, first = min(D.B, tid * per), last = min(D.B, first + per);
  uint64_t own = 0;
  bool any_bad = false, outside = false;
  for (uint32_t s = first; s < last; ++s) {
    PagedSeq q;
    bool bad;
    const int32_t c0 = cu[s], c1 = cu[s + 1], len = lens[s];
    if (s < kPagedHeld) {
      vm_paged_seq[0][s] = c0;
      vm_paged_seq[1][s] = c1;
      vm_paged_seq[2][s] = len;
    }
    if (paged_seq(D, c0, c1, len, &q, &bad)) {
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
  if ((tid & 63) == 63) vm_paged_cost[tid >> 6] = sum;
  any_bad = __syncthreads_or(any_bad);
  outside = __syncthreads_or(outside);
  auto uni64 = [](uint64_t x) { return (uint64_t(uni(uint32_t(x >> 32))) << 32) | uni(uint32_t(x)); };
  uint64_t before = sum - own, total = 0;
#pragma unroll
  for (uint32_t k = 0; k < uint32_t(kWaves); ++k) {
    if (k < (tid >> 6)) before += vm_paged_cost[k];
    total += vm_paged_cost[k];
  }
  total = uni64(total);
  if (any_bad || outside) paged_zero_rows(A, t, D, w, cu, lens, any_bad);
  w = uni(w);
  // a worker's share: share32 << sh, so that positions are divided by it in 32 bits
  const uint32_t bits = 64 - uint32_t(__builtin_clzll(total | 1)), sh = bits > 31 ? bits - 31 : 0;
  const uint32_t share32 = uni(max(max(kMinShare, min_share) >> min(sh, 20u), (uint32_t(total >> sh) + W) / W));
  const uint64_t share = uint64_t(share32) << sh;
  const uint64_t c0 = w * share, c1 = min(total, c0 + share);
  if (c0 >= total) return;
  // the sequence of cost c0
  if (own && before <= c0 && c0 < before + own) {
    uint64_t base = before;
    for (uint32_t s = first; s < last; ++s) {
      uint64_t c = own;
      if (per > 1) {
        PagedSeq q;
        bool bad;
        if (!paged_seq(D, cu[s], cu[s + 1], lens[s], &q, &bad)) continue;
        const PagedBlocks b = blocks(q);
        c = D.Hkv * b.before(b.nb);
      }
      if (c0 < base + c) {
        vm_paged_cost[kWaves] = base;
        vm_paged_cost[kWaves + 1] = s;
        break;
      }
      base += c;
    }
  }
  __syncthreads();
  uint64_t base = uni64(vm_paged_cost[kWaves]);
  uint32_t s = uni(uint32_t(vm_paged_cost[kWaves + 1]));

  uint32_t* arrivals = reinterpret_cast<uint32_t*>(A->scratch + A->task_scratch[ti]);
  float* scratch = reinterpret_cast<float*>(arrivals + kMaxLanes);
  const uint64_t slot_floats = paged_slot_floats(D);

  for (; s < D.B && base < c1; ++s) {
    PagedSeq q;
    if (!sequence(s, &q)) continue;
    const PagedBlocks B = blocks(q);
    const uint64_t S1 = B.before(B.nb);                        // a head's cost
    uint32_t h = 0, b = 0;
    uint64_t I0 = base;                                        // cost before the item
    if (c0 > base) {
      while (c0 - I0 >= S1) {                                  // at most Hkv - 1 times
        I0 += S1;
        ++h;
      }
      uint32_t hi = B.nb;                                      // the last b with before(b) <= c0 - I0
      while (hi - b > 1) {
        const uint32_t m = (b + hi) / 2;
        if (B.before(m) <= c0 - I0) b = m;
        else hi = m;
      }
      I0 += B.before(b);
    }
    for (; h < D.Hkv; ++h, b = 0) {
      bool done = false;
      for (; b < B.nb; ++b) {
        if (I0 >= c1) {
          done = true;
          break;
        }
        const uint32_t ks = B.kstart(b), K = B.kend(b) - ks;
        const uint64_t start = I0, I1 = I0 + kItemCost + uint64_t(K) * B.weight;
        I0 = I1;
        // Keys of the item before worker boundary c: a multiple of `align`, and none or all of
        // them where the boundary is nearer than `slack` to the item's start or end, since a
        // piece has to be worth its partial and the join (about 8 us for few rows, 20 for
        // many).  Where lanes are left over anyway (a share of less than 1024) an item of few
        // rows is cut later: alone it takes 10 us and 1.4 per 128 keys.  The boundaries between
        // give numbers that differ and are not 0, so that every piece counted below has keys:
        // a share and the slack are at least align * weight.
        const uint64_t slack = max(share < 1024 ? max(B.slack, 1024u) : B.slack, B.align * B.weight);
        const uint64_t from = start + kItemCost + slack, to = I1 > slack ? I1 - slack : 0;   // cut in (from, to)
        auto keys_before = [&](uint64_t c) -> uint32_t {
          if (c <= from) return 0;
          if (c >= to) return K;
          return uint32_t((c - start - kItemCost) / B.weight) / B.align * B.align;
        };
        const uint32_t ka = start >= c0 ? 0 : keys_before(c0), kb = I1 <= c1 ? K : keys_before(c1);
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
        uint32_t w0 = 0, np = 1;                              // worker of the first piece, pieces
        if (ka != 0 || kb != K) {
          // cut by the boundaries v * share in (from, to): w0 + 1, w0 + 2, ...
          w0 = uint32_t(from >> sh) / share32;
          while (uint64_t(w0 + 1) * share <= from) ++w0;
          uint32_t v = uint32_t((to - 1) >> sh) / share32;
          np = v - w0 + 1;
          job.part = scratch + (ka ? 2 * uint64_t(w) : 2 * uint64_t(w) + 1) * slot_floats;
        }
        if (body(job)) redo(job);
        if (!job.part) continue;
        // The barrier orders every thread's stores (done: vmcnt 0) before thread 0's arrival,
        // an agent-scope acquire-release that writes this XCD's L2 back, as at the grid
        // barrier; the last one sees every piece once its caches are invalidated.
        __builtin_amdgcn_s_waitcnt(0x0F70);
        __syncthreads();
        if (tid == 0) {
          const uint32_t n = __hip_atomic_fetch_add(arrivals + w0, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
          if (n == np - 1) __hip_atomic_store(arrivals + w0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          vm_paged_last = n == np - 1;
        }
        __syncthreads();
        if (vm_paged_last) {
          __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
          const uint32_t R = job.tokens * g;
          auto slot = [&](uint32_t i) -> const float* {
            return scratch + (i ? 2 * uint64_t(w0 + i) : 2 * uint64_t(w0) + 1) * slot_floats;
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
VM_LEAF void paged_block_generic(Args A, uint32_t ti, PagedJob J) {
  A = uargs(A);
  J.uniform();
  const VM_K Task& t = task_of(A, ti);
  const PagedDesc D = paged_desc(A, t);
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
      if (lane < hd / 8) {
        *(v4f*)(J.part + uint64_t(i) * hd + c) = v4f_make(o[0], o[1], o[2], o[3]);
        *(v4f*)(J.part + uint64_t(i) * hd + c + 4) = v4f_make(o[4], o[5], o[6], o[7]);
      }
      if (lane == 0) {
        J.part[uint64_t(R) * hd + i] = m;
        J.part[uint64_t(R) * (hd + 1) + i] = lsum;
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
    // a wave takes about 2 us for 64 keys of a row, of which a block has up to 32: 0.6 units
    // a key and row
    const uint32_t tb = max(1u, kPagedGenericRows / g);
    auto tokens = [&](uint32_t n, PagedBlocks* b) {
      const uint32_t rows = min(tb, n) * g;
      b->weight = min(32u, pow2_at_least(rows));
      b->align = 64;
      b->slack = 640;
      return tb;
    };
    paged_worker(A, ti, w, 2048, tokens, [&](const PagedJob& J) { return true; },
                 [&](const PagedJob& J) { paged_block_generic<DT, Q8>(A, ti, J); });
    __syncthreads();
  }
}

}  // namespace vm
