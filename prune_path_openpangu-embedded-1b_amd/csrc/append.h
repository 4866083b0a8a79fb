// What the appends to the paged caches, of 16 and of 8 bits, share: their arguments and the way of the heads that are
// normed and turned to rows of bfloat16.
#pragma once
#include "rotary.h"

#define APP_THREADS ROT_THREADS
#define APP_TOKENS 16

struct AppArgs {
  PagedSeqs seqs;
  const void *q, *k, *v;
  int64_t qs[2], ks[2], vs[2];  // strides of token and head, in elements
  bf16_t *q_out, *k_pages, *v_pages;
  const double* inv_freq;
  int Hq, Hkv, rd;
  float mscale;
  int zero_tail;
  int lgu, lgh;        // log2 of the threads on a head, and of rd / 2 (rounded up)
  int per, nqb, nkb;   // heads per block, blocks of query and of key heads
  int vper, nvb;       // the same of the value items
  uint32_t values;     // value items
};
// What only appends with norms, or to a cache of 8 bits, take besides.
struct AppMore {
  const void *qw, *kw;  // weights of the norms, NULL: none
  int w32;
  float eps;
  uint8_t *k8, *v8;     // the pages and scales (in place of k_pages and v_pages)
  uint8_t *k_scales, *v_scales;
};

// A unit's values, normed (lgu: log2 of the lanes on a head, all of the wave's taking part) and weighted.
template <typename T, bool HALF>
__device__ __forceinline__ void app_norm(const float (&wa)[8], const float (&wb)[8], int D, float eps, int lgu, float (&p)[8], float (&q)[8]) {
  const float2 r = head_scale<8>(p, q, head_sum(rot_squares<8>(p, q), lgu), D, eps, lgu);
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i] = p[i] * r.x * wa[i], q[i] = q[i] * r.x * wb[i];
}

// nt tokens (rows from `row` on, at positions from p0 on) of the nh query (kind 0) or key heads from h0 on, turned to y:
// token i, head h at y + i * yt + h * yh. `pair`, `freq`: the thread's pair of the table and its frequency, asked for
// by the caller. drop(): whether the tokens have no place.
template <typename T, int D, bool HALF, bool NORM, typename F>
__device__ __forceinline__ void app_turn(const AppArgs& a, const AppMore& e, int kind, float2* cs_s, double freq, int pair, int half, int64_t row, int nt,
                                         int h0, int nh, int64_t p0, bf16_t* y, int64_t yt, int64_t yh, F drop) {
  const int nr = half / 8, per = nr + (D - a.rd) / 8, tid = threadIdx.x;
  const RotLanes w(tid, a.lgu, 32 - __clz(nt - 1));  // as many tokens as there are
  const T* const x = (const T*)(kind == 0 ? a.q : a.k) + (row + w.i) * (kind == 0 ? a.qs[0] : a.ks[0]);
  const int64_t xs = kind == 0 ? a.qs[1] : a.ks[1];
  y += w.i * yt;
  int h = h0 + w.h;
  bool more = w.i < nt && h < h0 + nh && w.u < per;
  RotUnit<T, 8, HALF> now, next;
  float wa[8], wb[8];
  if constexpr (NORM) {
#pragma unroll
    for (int i = 0; i < 8; ++i) now.p.v[i] = now.q.v[i] = next.p.v[i] = next.q.v[i] = 0;
  }
  if (more) now.load(x + h * xs, w.u, nr, a.rd);
  if constexpr (NORM) rot_weights<8, HALF>(kind == 0 ? e.qw : e.kw, e.w32, w.u, nr, per, a.rd, wa, wb);
  paged_asked();
  if (pair < half)
    for (int t = tid >> a.lgh; t < nt; t += APP_THREADS >> a.lgh) cs_s[t * half + pair] = rot_entry(p0 + t, freq, a.mscale, 1.0f);
  if (drop()) return;
  __syncthreads();
  if constexpr (NORM) {
    for (int at = h0; at < h0 + nh; at += w.hstep) {  // (the folds need whole waves)
      const int h2 = h + w.hstep;
      const bool mine = more;
      more = more && h2 < h0 + nh;
      if (more) next.load(x + h2 * xs, w.u, nr, a.rd);
      float p[8], q[8];
      rot_pairs(now, w.u < nr, p, q);
      app_norm<T, HALF>(wa, wb, D, e.eps, a.lgu, p, q);
      if (mine) {
        if (w.u < nr) rot_turn<8>(cs_s + w.i * half + w.u * 8, p, q);
        rot_put<8, HALF>(y + h * yh, p, q, w.u, nr, a.rd);
      }
      now = next, h = h2;
    }
  } else {
    while (more) {
      const int h2 = h + w.hstep;
      more = h2 < h0 + nh;
      if (more) next.load(x + h2 * xs, w.u, nr, a.rd);
      now.store(y + h * yh, cs_s + w.i * half, w.u, nr, a.rd);
      now = next, h = h2;
    }
  }
}

// Of cache8.hip: the launch of an append to a cache of 8 bits, whose arguments have been checked.
int app8_launch(const char* what, AppArgs& a, const AppMore& e, int dtype, int D, int layout, int64_t n_tokens, hipStream_t stream);
