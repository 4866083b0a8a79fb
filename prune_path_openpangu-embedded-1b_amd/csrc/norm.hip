// Norms of queries and keys for each head, with the position rotation in the same pass, and their gradients.
//
//   x^ = x r,  r = 1 / sqrt(mean(x^2) + eps),  y = R (w x^)
//
// over the D channels of a head, R the turn of its first rotary_dim channels (rotary.h), w one weight a channel for
// all query heads and one for all key heads. With g = R^T dy (the turn by the opposite angles) and h = w g:
//
//   dw = sum over tokens and heads of g x^,   dx = r (h - x^ mean(h x^))
//
// A head lies in the registers of 2^lgu neighbouring lanes, one unit (V pairs, or V channels that are not turned) to
// each, so that both sums are folds over neighbours and x is read once. q and k go in one launch: a token's heads share
// its cos and sin. Everything between load and store is float32; one rounding.
//
// dw: a thread meets the same channels in every head, so it adds them up in registers over all that its workgroup
// takes, workgroups write one partial sum each, and a second launch adds those in order: the same bits every time.
//
// Memory bound: x and y once; x, dy and dx in the gradient. Queries and keys are launched as two sets of workgroups, each with
// its own weights (and their sums) in registers: with both sets in every thread, picked by the head, the backward took
// 221 registers, two waves a SIMD and 58 us for 8192 tokens of 24 bf16 heads of 128 (151 MB) where it now takes 32 (4.7 TB/s),
// the forward 26 where it takes 21 (101 MB, 4.8 TB/s, a large copy's rate), and the sums' launch 6.4 where it takes 3.8.
// float32, 3333 tokens of 24 heads of 80: 11.4 and 20.9 us (4.5 and 3.7 TB/s). One token: 3.4 us, a launch, its chain of
// loads and the sine.
#include <algorithm>
#include <cmath>

#include "rotary.h"

#define NORM_THREADS ROT_THREADS
#define NORM_MAX_D 256

// One of q and k in a launch: its workgroups are those from `first` on, gx groups of tokens by gy of heads.
struct NormSide {
  const void *x, *dy, *w;
  void* y;                // the result, or the gradient of x: [tokens][H][D]
  float* part;            // workspace: [gx * gy][D], NULL: no gradient of w
  int64_t xs[3], ds[3];   // strides of batch, token and head, in elements
  int H, lgt;             // heads, log2 of the tokens of a group
  uint32_t first, gx, gy;
};

struct NormArgs {
  NormSide side[2];
  const void* pos;
  const double* inv_freq;
  int64_t pb, pl;
  int64_t n;              // tokens
  uint32_t L;
  int D, rd, pos64, w32;
  float mscale, eps;
  int lgu, lgh;           // as in the rotation
};

// A lane's unit of a head. VEC: in 16-byte vectors; otherwise element by element, for any alignment and any even
// part that is turned, its last unit filled up with zeros.
template <typename T, int V, bool HALF, bool VEC>
struct NormUnit {
  RotUnit<T, V, HALF> x;
  // element i of the unit's first and second half in the head, -1: none
  static __device__ __forceinline__ int at(int i, bool second, int u, int nr, int half, int rd, int D) {
    if (u >= nr) return !second && rd + (u - nr) * V + i < D ? rd + (u - nr) * V + i : -1;
    const int j = u * V + i;
    return j >= half ? -1 : HALF ? j + (second ? half : 0) : 2 * j + second;
  }
  // `on`: whether there is a head, at p
  __device__ __forceinline__ void load(const T* p, bool on, int u, int nr, int per, int half, int rd, int D) {
#pragma unroll
    for (int i = 0; i < V; ++i) x.p.v[i] = x.q.v[i] = 0;
    if (!on || u >= per) return;
    if constexpr (VEC) x.load(p, u, nr, rd);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int j = at(i, false, u, nr, half, rd, D), k = at(i, true, u, nr, half, rd, D);
        if (j >= 0) x.p.v[i] = p[j];
        if (k >= 0) x.q.v[i] = p[k];
      }
  }
  __device__ __forceinline__ void pairs(bool turned, float (&a)[V], float (&b)[V]) const {
    if constexpr (VEC) rot_pairs(x, turned, a, b);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) a[i] = rot_f32(x.p.v[i]), b[i] = rot_f32(x.q.v[i]);
  }
  static __device__ __forceinline__ void put(T* y, const float (&a)[V], const float (&b)[V], int u, int nr, int half, int rd, int D) {
    if constexpr (VEC) rot_put<V, HALF>(y, a, b, u, nr, rd);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int j = at(i, false, u, nr, half, rd, D), k = at(i, true, u, nr, half, rd, D);
        const float one[1] = {a[i]}, two[1] = {b[i]};
        if (j >= 0) rot_store<1>(y + j, one);
        if (k >= 0) rot_store<1>(y + k, two);
      }
  }
  // the unit's weights
  static __device__ __forceinline__ void weights(const void* w, bool w32, int u, int nr, int per, int half, int rd, int D,
                                                 float (&a)[V], float (&b)[V]) {
    if constexpr (VEC) return rot_weights<V, HALF>(w, w32, u, nr, per, rd, a, b);
    int j[V], k[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      j[i] = u < per ? at(i, false, u, nr, half, rd, D) : -1, k[i] = u < per ? at(i, true, u, nr, half, rd, D) : -1;
    }
    if (w32) {  // the loads of one kind or of the other, without a branch between them
#pragma unroll
      for (int i = 0; i < V; ++i) a[i] = ((const float*)w)[max(j[i], 0)], b[i] = ((const float*)w)[max(k[i], 0)];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) a[i] = bf16_to_f32(((const bf16_t*)w)[max(j[i], 0)]), b[i] = bf16_to_f32(((const bf16_t*)w)[max(k[i], 0)]);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = j[i] < 0 ? 0.0f : a[i], b[i] = k[i] < 0 ? 0.0f : b[i];
  }
};

__device__ __forceinline__ int64_t norm_position(const NormArgs& a, uint32_t n) {
  const uint32_t b = n / a.L;
  const int64_t at = b * a.pb + (n - b * a.L) * a.pl;
  return a.pos64 ? ((const int64_t*)a.pos)[at] : (int64_t)((const int32_t*)a.pos)[at];
}

// What a workgroup has: a side, a group of tokens (the first of them, if it takes several) and a part of the heads.
template <typename F>
__device__ __forceinline__ void norm_work(const NormArgs& a, F f) {
  if (blockIdx.x < a.side[1].first) f(a.side[0], blockIdx.x);  // (one side's arguments at a time, in scalar registers)
  else f(a.side[1], blockIdx.x - a.side[1].first);
}

template <typename T, int V, bool HALF, bool VEC>
__global__ __launch_bounds__(NORM_THREADS) void qk_norm_kernel(NormArgs a) {
  using Unit = NormUnit<T, V, HALF, VEC>;
  __shared__ float2 cs_s[ROT_TABLE + V];  // (a unit that is not full reads past its token's last entry)
  const int half = a.rd / 2, nr = (half + V - 1) / V, per = nr + (a.D - a.rd + V - 1) / V, D = a.D, rd = a.rd;
  norm_work(a, [&](const NormSide& s, uint32_t id) {
    const uint32_t n0 = (id / s.gy) << s.lgt, gy = id % s.gy;
    const int nt = (int)min((uint32_t)1 << s.lgt, (uint32_t)a.n - n0);
    const RotLanes w(threadIdx.x, a.lgu, s.lgt);
    const int u = w.u, step = w.hstep * s.gy;
    const bool there = w.i < nt, turned = u < nr;
    const uint32_t n = n0 + (there ? w.i : 0), b = n / a.L, l = n - b * a.L;
    const T* const x = (const T*)s.x + b * s.xs[0] + l * s.xs[1];
    T* const y = (T*)s.y + (int64_t)n * s.H * D;
    int h = w.h + w.hstep * gy;
    Unit now, next;
    now.load(x + h * s.xs[2], there && h < s.H, u, nr, per, half, rd, D);
    float wa[V], wb[V];
    Unit::weights(s.w, a.w32, u, nr, per, half, rd, D, wa, wb);
    paged_asked();
    rot_table(cs_s, a.inv_freq, half, a.lgh, nt, a.mscale, 1.0f, [&](int t) { return norm_position(a, n0 + t); });
    __syncthreads();
    for (int h0 = w.hstep * gy; h0 < s.H; h0 += step, h += step) {  // (the folds need whole waves)
      next.load(x + (h + step) * s.xs[2], there && h + step < s.H, u, nr, per, half, rd, D);
      float p[V], q[V];
      now.pairs(turned, p, q);
      const float2 r = head_scale<V>(p, q, head_sum(rot_squares<V>(p, q), a.lgu), D, a.eps, a.lgu);
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = p[i] * r.x * wa[i], q[i] = q[i] * r.x * wb[i];
      if (there && h < s.H && u < per) {
        if (turned) rot_turn<V>(cs_s + w.i * half + u * V, p, q);
        Unit::put(y + h * D, p, q, u, nr, half, rd, D);
      }
      now = next;
    }
  });
}

template <typename T, int V, bool HALF, bool VEC>
__global__ __launch_bounds__(NORM_THREADS, VEC ? 4 : 2) void qk_norm_bwd_kernel(NormArgs a) {
  using Unit = NormUnit<T, V, HALF, VEC>;
  __shared__ float2 cs_s[ROT_TABLE + V];
  __shared__ float dw_s[NORM_THREADS / 64][NORM_MAX_D];
  const int half = a.rd / 2, nr = (half + V - 1) / V, per = nr + (a.D - a.rd + V - 1) / V, D = a.D, rd = a.rd;
  norm_work(a, [&](const NormSide& side, uint32_t id) {
    const uint32_t gy = id % side.gy;
    const RotLanes w(threadIdx.x, a.lgu, side.lgt);
    const int u = w.u, step = w.hstep * side.gy, H = side.H;
    const bool turned = u < nr;
    const float inv = 1.0f / D;
    float wa[V], wb[V], da[V], db[V];
    Unit::weights(side.w, a.w32, u, nr, per, half, rd, D, wa, wb);
#pragma unroll
    for (int i = 0; i < V; ++i) da[i] = db[i] = 0.0f;
    for (int64_t first = (int64_t)(id / side.gy) << side.lgt; first < a.n; first += (int64_t)side.gx << side.lgt) {
      const uint32_t n0 = (uint32_t)first;
      const int nt = (int)min((uint32_t)1 << side.lgt, (uint32_t)a.n - n0);
      const bool there = w.i < nt;
      const uint32_t n = n0 + (there ? w.i : 0), b = n / a.L, l = n - b * a.L;
      const T* const xp = (const T*)side.x + b * side.xs[0] + l * side.xs[1];
      const T* const gp = (const T*)side.dy + b * side.ds[0] + l * side.ds[1];
      T* const y = (T*)side.y + (int64_t)n * H * D;
      int h = w.h + w.hstep * gy;
      // (the next head's loads ahead of the present one's sums: 32 registers more, one wave of four less on a SIMD, and
      // 63 us instead of 60 for 8192 tokens of 24 heads with their forward)
      Unit x, g;
      auto load = [&](int h) {
        x.load(xp + h * side.xs[2], there && h < H, u, nr, per, half, rd, D);
        g.load(gp + h * side.ds[2], there && h < H, u, nr, per, half, rd, D);
      };
      load(h);
      __syncthreads();  // every thread is done with the entries before
      rot_table(cs_s, a.inv_freq, half, a.lgh, nt, a.mscale, -1.0f, [&](int t) { return norm_position(a, n0 + t); });
      __syncthreads();
      for (int h0 = w.hstep * gy; h0 < H; h0 += step, h += step) {
        float p[V], q[V], s[V], t[V];
        x.pairs(turned, p, q);
        g.pairs(turned, s, t);
        const bool on = there && h < H && u < per;
        if (on && turned) rot_turn<V>(cs_s + w.i * half + u * V, s, t);
        if constexpr (!VEC)  // what fills a unit up met no entry of its own
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (turned && u * V + i >= half) s[i] = t[i] = 0.0f;
        const float2 r = head_scale<V>(p, q, head_sum(rot_squares<V>(p, q), a.lgu), D, a.eps, a.lgu);
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          p[i] = on ? p[i] * r.x : 0.0f;
          q[i] = on ? q[i] * r.x : 0.0f;
          da[i] = __fmaf_rn(s[i], p[i], da[i]), db[i] = __fmaf_rn(t[i], q[i], db[i]);
          s[i] *= wa[i], t[i] *= wb[i];
          m = __fmaf_rn(s[i], p[i], __fmaf_rn(t[i], q[i], m));
        }
        m = head_sum(m, a.lgu) * inv;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          p[i] = __fmaf_rn(-p[i], m, s[i]) * r.x * r.y;
          q[i] = __fmaf_rn(-q[i], m, t[i]) * r.x * r.y;
        }
        if (on) Unit::put(y + h * D, p, q, u, nr, half, rd, D);
        load(h + step);
      }
    }
    if (!side.part) return;
    // the sums of a wave's lanes that meet the same channels, then of the waves
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < V; ++i)
      for (int m = 1 << a.lgu; m < 64; m <<= 1) {
        da[i] += __shfl_xor(da[i], m);
        db[i] += __shfl_xor(db[i], m);
      }
    if ((lane >> a.lgu) == 0 && u < per) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int j = Unit::at(i, false, u, nr, half, rd, D), k = Unit::at(i, true, u, nr, half, rd, D);
        if (j >= 0) dw_s[wave][j] = da[i];
        if (k >= 0) dw_s[wave][k] = db[i];
      }
    }
    __syncthreads();
    float* const to = side.part + (int64_t)id * D;
    for (int c = threadIdx.x; c < D; c += NORM_THREADS) to[c] = (dw_s[0][c] + dw_s[1][c]) + (dw_s[2][c] + dw_s[3][c]);
  });
}

// The workgroups' partial sums of either side added: 16 channels a workgroup (64 bytes of a row), 16 threads to each,
// which take rows in turn.
#define NORM_COLS 16
struct NormJoin {
  const float* part[2];
  void* dw[2];
  int rows[2];
  int D, w32;
};
__global__ __launch_bounds__(NORM_THREADS) void qk_norm_join_kernel(NormJoin a) {
  constexpr int G = NORM_THREADS / NORM_COLS, U = 8;
  __shared__ float sum_s[G][NORM_COLS];
  const int side = blockIdx.y, c = blockIdx.x * NORM_COLS + threadIdx.x % NORM_COLS, g = threadIdx.x / NORM_COLS, rows = a.rows[side];
  const float* const part = a.part[side] + min(c, a.D - 1);
  float s[U] = {};
  int i = g;
  for (; i + (U - 1) * G < rows; i += U * G)
#pragma unroll
    for (int j = 0; j < U; ++j) s[j] += part[(int64_t)(i + j * G) * a.D];
  for (; i < rows; i += G) s[0] += part[(int64_t)i * a.D];
  sum_s[g][threadIdx.x % NORM_COLS] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  if (g || c >= a.D || !a.dw[side]) return;
  float t = 0.0f;
#pragma unroll
  for (int k = 0; k < G; ++k) t += sum_s[k][threadIdx.x];
  if (a.w32) ((float*)a.dw[side])[c] = t;
  else ((bf16_t*)a.dw[side])[c] = f32_to_bf16(t);
}

// ------------------------------------------------------------------ host
// Sizes that the launch of one side, and the workspace of the gradient, go by.
struct NormPlan {
  int lgt;
  int64_t gx, gy;
};

static NormPlan norm_plan(int64_t n, int H, int D, int rd, int V, bool backward) {
  NormPlan p = {};
  if (H == 0) return p;
  const int half = rd / 2, per = (half + V - 1) / V + (D - rd + V - 1) / V, lgu = rot_log2up(per);
  const int64_t cus = pp_device_cus();
  while (p.lgt < 4 && lgu + p.lgt < 8 && ((int64_t)H * per << p.lgt) < 4 * NORM_THREADS && (n >> (p.lgt + 1)) >= 2 * cus &&
         (half << (p.lgt + 1)) <= ROT_TABLE)
    ++p.lgt;
  const int64_t groups = (n + (1 << p.lgt) - 1) >> p.lgt, hstep = (NORM_THREADS >> lgu) >> p.lgt;
  p.gx = backward ? std::min<int64_t>(groups, 2 * cus) : groups;
  p.gy = std::max<int64_t>(1, std::min<int64_t>((H + hstep - 1) / hstep, (2 * cus + p.gx - 1) / p.gx));
  return p;
}

static int norm_sizes(const char* what, int dtype, int64_t batch, int64_t length, int Hq, int Hk, int D, int rotary_dim) {
  PP_REQUIRE(dtype == PP_DTYPE_F32 || dtype == PP_DTYPE_BF16, PP_ERR_INVALID, "%s: dtype %d", what, dtype);
  PP_REQUIRE(D >= 2 && D <= NORM_MAX_D, PP_ERR_UNSUPPORTED, "%s: head size %d unsupported (2..%d)", what, D, NORM_MAX_D);
  PP_REQUIRE(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= D, PP_ERR_INVALID,
             "%s: rotary_dim %d (need an even number, 2 to the head size %d)", what, rotary_dim, D);
  PP_REQUIRE(batch >= 0 && length >= 0 && Hq >= 0 && Hk >= 0 && Hq <= 65536 && Hk <= 65536 && batch <= 0x7fffffff &&
                 length <= 0x7fffffff && batch * length <= 0x7fffffff,
             PP_ERR_UNSUPPORTED, "%s: %lld x %lld tokens of %d and %d heads", what, (long long)batch, (long long)length, Hq, Hk);
  return PP_OK;
}

// float32 in units of 4 (16 bytes), unless a head then takes more than a wave's lanes
static int norm_unit(int dtype, int D, int rd) {
  return dtype == PP_DTYPE_F32 && (rd / 2 + 3) / 4 + (D - rd + 3) / 4 <= 64 ? 4 : 8;
}

static int norm_launch(const char* what, NormArgs& a, int dtype, int layout, bool backward, bool vec, int V, hipStream_t st) {
  int64_t groups = 0;
  for (int i = 0; i < 2; ++i) {
    const NormPlan p = norm_plan(a.n, a.side[i].H, a.D, a.rd, V, backward);
    a.side[i].lgt = p.lgt, a.side[i].gx = (uint32_t)p.gx, a.side[i].gy = (uint32_t)std::max<int64_t>(p.gy, 1);
    a.side[i].first = (uint32_t)groups;
    groups += p.gx * p.gy;
    PP_REQUIRE(groups <= 0xffffff, PP_ERR_UNSUPPORTED, "%s: %lld tokens of this head size", what, (long long)a.n);
  }
  a.lgu = rot_log2up((a.rd / 2 + V - 1) / V + (a.D - a.rd + V - 1) / V), a.lgh = std::min(8, rot_log2up(a.rd / 2));
  const unsigned grid = (unsigned)groups;
#define NORM(T, V_, HALF_, VEC_)                                                                 \
  do {                                                                                           \
    if (backward) qk_norm_bwd_kernel<T, V_, HALF_, VEC_><<<grid, NORM_THREADS, 0, st>>>(a);      \
    else qk_norm_kernel<T, V_, HALF_, VEC_><<<grid, NORM_THREADS, 0, st>>>(a);                   \
  } while (0)
#define NORM_LAYOUT(T, V_, VEC_)                           \
  do {                                                     \
    if (layout == PP_ROTARY_HALF) NORM(T, V_, true, VEC_); \
    else NORM(T, V_, false, VEC_);                         \
  } while (0)
  if (dtype == PP_DTYPE_F32) {
    if (vec) NORM_LAYOUT(float, 4, true);
    else if (V == 4) NORM_LAYOUT(float, 4, false);
    else NORM_LAYOUT(float, 8, false);
  } else {
    if (vec) NORM_LAYOUT(bf16_t, 8, true);
    else NORM_LAYOUT(bf16_t, 8, false);
  }
#undef NORM_LAYOUT
#undef NORM
  return pp_check_launch(what);
}

static int norm_args(const char* what, NormArgs& a, int w_dtype, const void* positions, int pos64, const int64_t* pos_strides,
                     int64_t batch, int64_t length, int Hq, int Hk, int D, const double* inv_freq, int rotary_dim, int layout,
                     float mscale, float eps, int dtype) {
  PP_REQUIRE(layout == PP_ROTARY_HALF || layout == PP_ROTARY_INTERLEAVED, PP_ERR_INVALID, "%s: layout %d", what, layout);
  PP_REQUIRE(w_dtype == dtype || w_dtype == PP_DTYPE_F32, PP_ERR_INVALID, "%s: weights of dtype %d for heads of %d", what, w_dtype, dtype);
  PP_REQUIRE(eps >= 0.0f && std::isfinite(eps), PP_ERR_INVALID, "%s: eps %g", what, eps);
  PP_REQUIRE(positions && pos_strides && inv_freq, PP_ERR_INVALID, "%s: null pointer", what);
  a.pos = positions, a.pos64 = pos64, a.pb = pos_strides[0], a.pl = pos_strides[1];
  a.inv_freq = inv_freq, a.n = batch * length, a.L = (uint32_t)length, a.side[0].H = Hq, a.side[1].H = Hk;
  a.D = D, a.rd = rotary_dim, a.w32 = w_dtype == PP_DTYPE_F32, a.mscale = mscale, a.eps = eps;
  return PP_OK;
}

extern "C" int pp_qk_norm_rotary(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, int dtype,
                                 const void* q_weight, const void* k_weight, int w_dtype, const void* positions, int pos64,
                                 const int64_t* pos_strides, int64_t batch, int64_t length, int Hq, int Hk, int D,
                                 const double* inv_freq, int rotary_dim, int layout, float mscale, float eps, void* q_out,
                                 void* k_out, void* stream) {
  const char* const what = "pp_qk_norm_rotary";
  int rc = norm_sizes(what, dtype, batch, length, Hq, Hk, D, rotary_dim);
  if (rc || batch == 0 || length == 0 || Hq + Hk == 0) return rc;
  NormArgs a = {};
  rc = norm_args(what, a, w_dtype, positions, pos64, pos_strides, batch, length, Hq, Hk, D, inv_freq, rotary_dim, layout, mscale, eps, dtype);
  if (rc) return rc;
  PP_REQUIRE((Hq == 0 || (q && q_strides && q_weight && q_out)) && (Hk == 0 || (k && k_strides && k_weight && k_out)), PP_ERR_INVALID,
             "%s: null pointer", what);
  const int bytes = dtype == PP_DTYPE_F32 ? 4 : 2, V = norm_unit(dtype, D, rotary_dim);
  bool vec = V * bytes == 16 && (rotary_dim / 2) % V == 0 && (D - rotary_dim) % V == 0;
  const void *xs[2] = {q, k}, *ws[2] = {q_weight, k_weight};
  void* ys[2] = {q_out, k_out};
  const int64_t* ss[2] = {q_strides, k_strides};
  for (int i = 0; i < 2; ++i) {
    NormSide& s = a.side[i];
    if (s.H == 0) continue;
    s.x = xs[i], s.y = ys[i], s.w = ws[i];
    for (int j = 0; j < 3; ++j) s.xs[j] = ss[i][j];
    vec = vec && ((uintptr_t)ws[i] & 15) == 0 && rot_aligned(xs[i], ss[i], 3, bytes) && ((uintptr_t)ys[i] & 15) == 0;
  }
  return norm_launch(what, a, dtype, layout, false, vec, V, (hipStream_t)stream);
}

extern "C" size_t pp_qk_norm_rotary_workspace_bytes(int dtype, int64_t batch, int64_t length, int Hq, int Hk, int D, int rotary_dim) {
  if (norm_sizes("pp_qk_norm_rotary_bwd", dtype, batch, length, Hq, Hk, D, rotary_dim)) return 0;
  if (batch == 0 || length == 0 || Hq + Hk == 0) return 0;
  const int V = norm_unit(dtype, D, rotary_dim);
  const NormPlan p = norm_plan(batch * length, Hq, D, rotary_dim, V, true), q = norm_plan(batch * length, Hk, D, rotary_dim, V, true);
  return (size_t)(p.gx * p.gy + q.gx * q.gy) * D * 4;
}

extern "C" int pp_qk_norm_rotary_bwd(const void* dq, const int64_t* dq_strides, const void* dk, const int64_t* dk_strides,
                                     const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, int dtype,
                                     const void* q_weight, const void* k_weight, int w_dtype, const void* positions, int pos64,
                                     const int64_t* pos_strides, int64_t batch, int64_t length, int Hq, int Hk, int D,
                                     const double* inv_freq, int rotary_dim, int layout, float mscale, float eps, void* q_grad,
                                     void* k_grad, void* q_weight_grad, void* k_weight_grad, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  const char* const what = "pp_qk_norm_rotary_bwd";
  int rc = norm_sizes(what, dtype, batch, length, Hq, Hk, D, rotary_dim);
  if (rc) return rc;
  PP_REQUIRE(w_dtype == PP_DTYPE_F32 || w_dtype == PP_DTYPE_BF16, PP_ERR_INVALID, "%s: weights of dtype %d", what, w_dtype);
  const bool need = q_weight_grad || k_weight_grad;
  hipStream_t st = (hipStream_t)stream;
  const dim3 joins((D + NORM_COLS - 1) / NORM_COLS, 2);
  NormJoin join = {{nullptr, nullptr}, {q_weight_grad, k_weight_grad}, {0, 0}, D, w_dtype == PP_DTYPE_F32};
  if (batch == 0 || length == 0 || Hq + Hk == 0) {  // a sum of nothing
    if (need) qk_norm_join_kernel<<<joins, NORM_THREADS, 0, st>>>(join);
    return need ? pp_check_launch(what) : PP_OK;
  }
  NormArgs a = {};
  rc = norm_args(what, a, w_dtype, positions, pos64, pos_strides, batch, length, Hq, Hk, D, inv_freq, rotary_dim, layout, mscale, eps, dtype);
  if (rc) return rc;
  PP_REQUIRE((Hq == 0 || (dq && dq_strides && q && q_strides && q_weight && q_grad)) &&
                 (Hk == 0 || (dk && dk_strides && k && k_strides && k_weight && k_grad)),
             PP_ERR_INVALID, "%s: null pointer", what);
  const int bytes = dtype == PP_DTYPE_F32 ? 4 : 2, V = norm_unit(dtype, D, rotary_dim);
  bool vec = V * bytes == 16 && (rotary_dim / 2) % V == 0 && (D - rotary_dim) % V == 0;
  const void *xs[2] = {q, k}, *gs[2] = {dq, dk}, *ws[2] = {q_weight, k_weight};
  void* ys[2] = {q_grad, k_grad};
  const int64_t *ss[2] = {q_strides, k_strides}, *ds[2] = {dq_strides, dk_strides};
  for (int i = 0; i < 2; ++i) {
    NormSide& s = a.side[i];
    if (s.H == 0) continue;
    s.x = xs[i], s.dy = gs[i], s.y = ys[i], s.w = ws[i];
    for (int j = 0; j < 3; ++j) s.xs[j] = ss[i][j], s.ds[j] = ds[i][j];
    vec = vec && ((uintptr_t)ws[i] & 15) == 0 && rot_aligned(xs[i], ss[i], 3, bytes) && rot_aligned(gs[i], ds[i], 3, bytes) && ((uintptr_t)ys[i] & 15) == 0;
  }
  const NormPlan p[2] = {norm_plan(a.n, Hq, D, rotary_dim, V, true), norm_plan(a.n, Hk, D, rotary_dim, V, true)};
  for (int i = 0; i < 2; ++i) join.rows[i] = (int)(p[i].gx * p[i].gy);
  const size_t bytes_needed = need ? (size_t)(join.rows[0] + join.rows[1]) * D * 4 : 0;
  PP_REQUIRE(bytes_needed == 0 || (workspace && workspace_bytes >= bytes_needed && ((uintptr_t)workspace & 15) == 0), PP_ERR_INVALID,
             "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", what, workspace_bytes, bytes_needed);
  if (need) {
    a.side[0].part = (float*)workspace, a.side[1].part = a.side[0].part + (size_t)join.rows[0] * D;
    join.part[0] = a.side[0].part, join.part[1] = a.side[1].part;
  }
  rc = norm_launch(what, a, dtype, layout, true, vec, V, st);
  if (rc || !need) return rc;
  qk_norm_join_kernel<<<joins, NORM_THREADS, 0, st>>>(join);
  return pp_check_launch(what);
}
