// What the kernels that turn heads by their positions share: cos and sin of a workgroup's tokens in LDS, a thread's
// unit of a head, the workgroup's threads on units, tokens and heads.
#pragma once
#include "paged.h"

#define ROT_THREADS 256
#define ROT_TABLE 2048  // (cos, sin) entries in LDS

// V consecutive elements as they are in memory (more than one: in 16-byte words)
template <typename T, int V>
struct RotPack {
  T v[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 1) v[0] = *p;
    else *this = *(const RotPack*)__builtin_assume_aligned(p, 16);
  }
};
__device__ __forceinline__ float rot_f32(float x) { return x; }
__device__ __forceinline__ float rot_f32(bf16_t x) { return bf16_to_f32(x); }
template <int V>
__device__ __forceinline__ void rot_store(float* p, const float (&v)[V]) {
  if constexpr (V == 1) *p = v[0];
  else
#pragma unroll
    for (int i = 0; i < V; i += 4) *(float4*)(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}
template <int V>
__device__ __forceinline__ void rot_store(bf16_t* p, const float (&v)[V]) {
  if constexpr (V == 8)
    *(uint4*)p = make_uint4(f32_to_bf16x2(v[0], v[1]), f32_to_bf16x2(v[2], v[3]), f32_to_bf16x2(v[4], v[5]), f32_to_bf16x2(v[6], v[7]));
  else
    *p = f32_to_bf16(v[0]);
}

// (m cos a, m sin a) of a = position * inv_freq
__device__ __forceinline__ float2 rot_entry(int64_t position, double inv_freq, float m, float sign) {
  const double turns = (double)position * (inv_freq * 0.15915494309189533577);
  const double exact = 2.0 * (turns - rint(turns));
  const float half_turns = (float)exact, left = (float)((exact - half_turns) * 3.14159265358979323846);
  float s, c;
  sincospif(half_turns, &s, &c);
  return make_float2(__fmaf_rn(-s, left, c) * m, sign * __fmaf_rn(c, left, s) * m);
}

// A unit of a head: u < nr turns V pairs, the units behind them copy V channels. Its loads apart from
// the rest, so that they are on their way while cos and sin are computed.
template <typename TI, int V, bool HALF>
struct RotUnit {
  RotPack<TI, V> p, q;
  __device__ __forceinline__ void load(const TI* x, int u, int nr, int rd) {
    if (u < nr) {
      const int a = HALF ? u * V : 2 * u * V, b = HALF ? rd / 2 + u * V : a + V;
      p.load(x + a);
      q.load(x + b);
    } else
      p.load(x + rd + (u - nr) * V);
  }
  template <typename TO>
  __device__ __forceinline__ void store(TO* y, const float2* cs, int u, int nr, int rd) const {
    float r[V], t[V];
    if (u < nr) {
      const int a = HALF ? u * V : 2 * u * V, b = HALF ? rd / 2 + u * V : a + V;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        // the pair: one of p and one of q, or two neighbours of what p and q hold together
        const float x1 = rot_f32(HALF ? p.v[i] : 2 * i < V ? p.v[2 * i % V] : q.v[2 * i % V]);
        const float x2 = rot_f32(HALF ? q.v[i] : 2 * i + 1 < V ? p.v[(2 * i + 1) % V] : q.v[(2 * i + 1) % V]);
        const float2 w = cs[u * V + i];
        const float y1 = __fmaf_rn(x1, w.x, -__fmul_rn(x2, w.y)), y2 = __fmaf_rn(x1, w.y, __fmul_rn(x2, w.x));
        if (HALF) {
          r[i] = y1, t[i] = y2;
        } else {
          (2 * i < V ? r : t)[2 * i % V] = y1;
          (2 * i + 1 < V ? r : t)[(2 * i + 1) % V] = y2;
        }
      }
      rot_store<V>(y + a, r);
      rot_store<V>(y + b, t);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) r[i] = rot_f32(p.v[i]);
      rot_store<V>(y + rd + (u - nr) * V, r);
      asm volatile("");  // the two sides' last stores, merged, went out as 4 and 12 bytes
    }
  }
};

// The unit's values as pairs, and a unit's pairs to memory: b is 0, and not stored, in a unit that is copied.
template <typename TI, int V, bool HALF>
__device__ __forceinline__ void rot_pairs(const RotUnit<TI, V, HALF>& x, bool turned, float (&a)[V], float (&b)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float one = rot_f32(x.p.v[i]);
    if (HALF) {
      a[i] = one, b[i] = turned ? rot_f32(x.q.v[i]) : 0.0f;
    } else {
      const float x1 = rot_f32(2 * i < V ? x.p.v[2 * i % V] : x.q.v[2 * i % V]);
      const float x2 = rot_f32(2 * i + 1 < V ? x.p.v[(2 * i + 1) % V] : x.q.v[(2 * i + 1) % V]);
      a[i] = turned ? x1 : one, b[i] = turned ? x2 : 0.0f;
    }
  }
}
template <int V, bool HALF, typename TO>
__device__ __forceinline__ void rot_put(TO* y, const float (&a)[V], const float (&b)[V], int u, int nr, int rd) {
  if (u < nr) {
    if (HALF) {
      rot_store<V>(y + u * V, a);
      rot_store<V>(y + rd / 2 + u * V, b);
    } else {
      float r[V], t[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        (2 * i < V ? r : t)[2 * i % V] = a[i];
        (2 * i + 1 < V ? r : t)[(2 * i + 1) % V] = b[i];
      }
      rot_store<V>(y + 2 * u * V, r);
      rot_store<V>(y + 2 * u * V + V, t);
    }
  } else {
    rot_store<V>(y + rd + (u - nr) * V, a);
    asm volatile("");  // as above
  }
}
// (a, b) turned by the entries of cs
template <int V>
__device__ __forceinline__ void rot_turn(const float2* cs, float (&a)[V], float (&b)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float2 w = cs[i];
    const float y1 = __fmaf_rn(a[i], w.x, -__fmul_rn(b[i], w.y)), y2 = __fmaf_rn(a[i], w.y, __fmul_rn(b[i], w.x));
    a[i] = y1, b[i] = y2;
  }
}

// ------------------------------------------------------------------ norms of heads
// The weights of a unit's channels, from a row that starts on a 16-byte boundary: float32, or bfloat16.
template <int V, bool HALF>
__device__ __forceinline__ void rot_weights(const void* w, bool w32, int u, int nr, int per, int rd, float (&a)[V], float (&b)[V]) {
  const int at = min(u, per - 1);
  if (w32) {
    RotUnit<float, V, HALF> x;
    x.load((const float*)w, at, nr, rd);
    rot_pairs(x, at < nr, a, b);
  } else if constexpr (V == 8) {
    RotUnit<bf16_t, V, HALF> x;
    x.load((const bf16_t*)w, at, nr, rd);
    rot_pairs(x, at < nr, a, b);
  }
}
// A reduction over the 2^lgu neighbours that hold a head, in every one of them; every lane of the wave takes part.
template <typename F>
__device__ __forceinline__ float head_fold(float v, int lgu, F f) {
  const int lane = threadIdx.x & 63;
  if (lgu > 0) v = f(v, dpp_mov<PP_DPP_XOR1>(v));
  if (lgu > 1) v = f(v, dpp_mov<PP_DPP_XOR2>(v));
  if (lgu > 2) v = f(v, dpp_mov<PP_DPP_HALF_MIRROR>(v));
  if (lgu > 3) v = f(v, dpp_mov<PP_DPP_ROR8>(v));
  if (lgu > 4) v = f(v, pl_xor16f(v, lane));
  if (lgu > 5) v = f(v, pl_xor32f(v, lane));
  return v;
}
__device__ __forceinline__ float head_sum(float v, int lgu) {
  return head_fold(v, lgu, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float head_max(float v, int lgu) {
  return head_fold(v, lgu, [](float a, float b) { return fmaxf(a, b); });
}
template <int V>
__device__ __forceinline__ float rot_squares(const float (&a)[V], const float (&b)[V]) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) s = __fmaf_rn(a[i], a[i], __fmaf_rn(b[i], b[i], s));
  return s;
}
// What a head's values are to be multiplied by: x of the result, 1 / sqrt(mean of squares + eps). ss: the head's sum of
// squares. If the squares leave float32's range, the values are first multiplied, here, by what brings the largest of
// them next to 1, y of the result, and x is that of these.
template <int V>
__device__ __forceinline__ float2 head_scale(float (&a)[V], float (&b)[V], float ss, int D, float eps, int lgu) {
  const float inv = 1.0f / D, mean = __fmaf_rn(ss, inv, eps);
  float r = rsqrtf(mean), pre = 1.0f;
  const bool odd = !(mean >= 0x1p-100f && ss <= 0x1p120f);
  if (__builtin_expect(__ballot(odd) != 0, 0)) {  // the whole wave: the folds below need its lanes
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) top = fmaxf(top, fmaxf(fabsf(a[i]), fabsf(b[i])));
    top = head_max(top, lgu);
    const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -126), 126);
    const float by = __uint_as_float((uint32_t)(127 - e) << 23);
    float x[V], y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = a[i] * by, y[i] = b[i] * by;
    const float ss2 = head_sum(rot_squares<V>(x, y), lgu), e2 = eps * by * by;
    if (odd && top > 0.0f && top < __builtin_inff()) {
      pre = by;
      r = e2 < __builtin_inff() ? rsqrtf(__fmaf_rn(ss2, inv, e2)) : rsqrtf(eps) / by;
#pragma unroll
      for (int i = 0; i < V; ++i) a[i] = x[i], b[i] = y[i];
    }
  }
  return make_float2(r, pre);
}

// A workgroup's threads: 2^lgu neighbours on the units of a head, then 2^lgt tokens, then heads; all by
// shifts (divisions cost more than the turning).
struct RotLanes {
  int u, i, h, hstep;
  __device__ RotLanes(int tid, int lgu, int lgt) {
    u = tid & ((1 << lgu) - 1);
    i = (tid >> lgu) & ((1 << lgt) - 1);
    h = tid >> (lgu + lgt);
    hstep = (ROT_THREADS >> lgu) >> lgt;
  }
};
static inline int rot_log2up(int64_t v) {
  int b = 0;
  while (((int64_t)1 << b) < v) ++b;
  return b;
}

// cos and sin of nt tokens into LDS, position(t) theirs
template <typename F>
__device__ __forceinline__ void rot_table(float2* cs, const double* inv_freq, int half, int lgh, int nt, float m, float sign,
                                          F position) {
  for (int f = threadIdx.x & ((1 << lgh) - 1); f < half; f += ROT_THREADS)  // once, unless there are more than threads
    for (int t = threadIdx.x >> lgh; t < nt; t += max(ROT_THREADS >> lgh, 1))
      cs[t * half + f] = rot_entry(position(t), inv_freq[f], m, sign);
}

static inline bool rot_aligned(const void* p, const int64_t* s, int n, int bytes) {
  bool ok = ((uintptr_t)p & 15) == 0;
  for (int i = 0; i < n; ++i) ok = ok && (s[i] * bytes) % 16 == 0;
  return ok;
}
