// Rotary positions, and the append of keys and values to a paged cache with the rotation on the way.
//
// Pair i of a head (of the first rotary_dim channels) turns by the angle a = position * inv_freq[i]:
//   y1 = m (x1 cos a - x2 sin a),  y2 = m (x1 sin a + x2 cos a)
// (x1, x2) = channels (i, rotary_dim / 2 + i) in the half layout, (2 i, 2 i + 1) interleaved; the
// channels from rotary_dim on are copied. The transpose, which is the gradient's map, is the turn
// by -a with the same m.
//
// The angle is taken in turns: position * (inv_freq / 2 pi) as a float64 product, of which only the
// part beyond the nearest whole turn goes to float32. In float32 the product itself would be off by
// 2^-24 of the angle: 0.06 rad at a million radians.
//
// Memory bound: one read, one write. cos and sin of a workgroup's tokens are computed once into
// LDS, then its threads stream the tokens' heads in 16-byte vectors, 8 pairs a step.
#include <algorithm>

#include "paged.h"

#define ROT_THREADS 256
#define ROT_TABLE 2048  // (cos, sin) entries in LDS

typedef uint32_t rot_u4 __attribute__((ext_vector_type(4)));

// V consecutive elements as floats (V = 8: 16-byte vectors)
template <typename T, int V>
struct RotVec;
template <>
struct RotVec<float, 8> {
  static __device__ __forceinline__ void load(const float* p, float (&v)[8]) {
    const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[8]) {
    *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
    *(float4*)(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  }
};
template <>
struct RotVec<bf16_t, 8> {
  static __device__ __forceinline__ void load(const bf16_t* p, float (&v)[8]) {
    const uint4 u = *(const uint4*)p;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store(bf16_t* p, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = f32_to_bf16x2(v[2 * i], v[2 * i + 1]);
    *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct RotVec<float, 1> {
  static __device__ __forceinline__ void load(const float* p, float (&v)[1]) { v[0] = *p; }
  static __device__ __forceinline__ void store(float* p, const float (&v)[1]) { *p = v[0]; }
};
template <>
struct RotVec<bf16_t, 1> {
  static __device__ __forceinline__ void load(const bf16_t* p, float (&v)[1]) { v[0] = bf16_to_f32(*p); }
  static __device__ __forceinline__ void store(bf16_t* p, const float (&v)[1]) { *p = f32_to_bf16(v[0]); }
};

// (m cos a, m sin a) of a = position * inv_freq
__device__ __forceinline__ float2 rot_entry(int64_t position, double inv_freq, float m, float sign) {
  const double turns = (double)position * (inv_freq * 0.15915494309189533577);
  const float half_turns = (float)(2.0 * (turns - rint(turns)));
  float s, c;
  sincospif(half_turns, &s, &c);
  return make_float2(c * m, sign * s * m);
}

// One step of a head: unit u < nr turns V pairs, the units behind them copy V channels.
template <typename TI, typename TO, int V, bool HALF>
__device__ __forceinline__ void rot_unit(const TI* x, TO* y, const float2* cs, int u, int nr, int rd) {
  if (u < nr) {
    const int a = HALF ? u * V : 2 * u * V, b = HALF ? rd / 2 + u * V : a + V;
    float p[V], q[V], r[V], t[V];
    RotVec<TI, V>::load(x + a, p);
    RotVec<TI, V>::load(x + b, q);
    if (HALF) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 w = cs[u * V + i];
        r[i] = __fmaf_rn(p[i], w.x, -__fmul_rn(q[i], w.y));
        t[i] = __fmaf_rn(p[i], w.y, __fmul_rn(q[i], w.x));
      }
    } else {
      float in[2 * V], out[2 * V];
#pragma unroll
      for (int i = 0; i < V; ++i) in[i] = p[i], in[V + i] = q[i];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 w = cs[u * V + i];
        out[2 * i] = __fmaf_rn(in[2 * i], w.x, -__fmul_rn(in[2 * i + 1], w.y));
        out[2 * i + 1] = __fmaf_rn(in[2 * i], w.y, __fmul_rn(in[2 * i + 1], w.x));
      }
#pragma unroll
      for (int i = 0; i < V; ++i) r[i] = out[i], t[i] = out[V + i];
    }
    RotVec<TO, V>::store(y + a, r);
    RotVec<TO, V>::store(y + b, t);
  } else {
    float p[V];
    const int a = rd + (u - nr) * V;
    RotVec<TI, V>::load(x + a, p);
    RotVec<TO, V>::store(y + a, p);
  }
}

struct RotArgs {
  const void* x;
  void* y;
  const void* pos;
  const double* inv_freq;
  int64_t xs[3], ys[3];  // strides of batch, token and head, in elements
  int64_t pb, pl;        // strides of the positions
  int64_t n;             // tokens
  uint32_t L, heads;
  int D, rd, pos64;
  float mscale, sign;
  int tokens;            // per workgroup
};

template <typename T, int V, bool HALF>
__global__ __launch_bounds__(ROT_THREADS) void rotary_kernel(RotArgs a) {
  __shared__ float2 cs_s[ROT_TABLE];
  const int tid = threadIdx.x, half = a.rd / 2;
  const int64_t n0 = (int64_t)blockIdx.x * a.tokens;
  const int nt = (int)min((int64_t)a.tokens, a.n - n0);
  for (int k = tid; k < nt * half; k += ROT_THREADS) {
    const int t = k / half;
    const int64_t n = n0 + t, b = n / a.L, l = n - b * a.L;
    const int64_t at = b * a.pb + l * a.pl;
    const int64_t p = a.pos64 ? ((const int64_t*)a.pos)[at] : (int64_t)((const int32_t*)a.pos)[at];
    cs_s[k] = rot_entry(p, a.inv_freq[k - t * half], a.mscale, a.sign);
  }
  __syncthreads();
  const uint32_t nr = half / V, per = nr + (a.D - a.rd) / V, units = a.heads * per;
  for (uint32_t k = blockIdx.y * ROT_THREADS + tid; k < nt * units; k += gridDim.y * ROT_THREADS) {
    const uint32_t t = k / units, r = k - t * units, h = r / per, u = r - h * per;
    const int64_t n = n0 + t, b = n / a.L, l = n - b * a.L;
    rot_unit<T, T, V, HALF>((const T*)a.x + b * a.xs[0] + l * a.xs[1] + h * a.xs[2],
                            (T*)a.y + b * a.ys[0] + l * a.ys[1] + h * a.ys[2], cs_s + t * half, u, nr, a.rd);
  }
}

static bool rot_aligned(const void* p, const int64_t* s, int n, int bytes) {
  bool ok = ((uintptr_t)p & 15) == 0;
  for (int i = 0; i < n; ++i) ok = ok && (s[i] * bytes) % 16 == 0;
  return ok;
}

extern "C" int pp_rotary(const void* x, int dtype, const int64_t* x_strides, const void* positions, int pos64,
                         const int64_t* pos_strides, int64_t batch, int64_t length, int heads, int D,
                         const double* inv_freq, int rotary_dim, int layout, float mscale, int inverse, void* y,
                         const int64_t* y_strides, void* stream) {
  const char* const what = "pp_rotary";
  PP_REQUIRE(dtype == PP_DTYPE_F32 || dtype == PP_DTYPE_BF16, PP_ERR_INVALID, "%s: dtype %d", what, dtype);
  PP_REQUIRE(layout == PP_ROTARY_HALF || layout == PP_ROTARY_INTERLEAVED, PP_ERR_INVALID, "%s: layout %d", what, layout);
  PP_REQUIRE(D >= 1 && D <= 1024, PP_ERR_UNSUPPORTED, "%s: head size %d unsupported (1..1024)", what, D);
  PP_REQUIRE(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= D, PP_ERR_INVALID,
             "%s: rotary_dim %d (need an even number, 2 to the head size %d)", what, rotary_dim, D);
  PP_REQUIRE(batch >= 0 && length >= 0 && heads >= 0 && heads <= 65536 && batch <= 0x7fffffff && length <= 0x7fffffff &&
                 batch * length <= 0x7fffffff,
             PP_ERR_UNSUPPORTED, "%s: %lld x %lld tokens of %d heads", what, (long long)batch, (long long)length, heads);
  if (batch == 0 || length == 0 || heads == 0) return PP_OK;
  PP_REQUIRE(x && positions && inv_freq && y && x_strides && y_strides && pos_strides, PP_ERR_INVALID,
             "%s: null pointer", what);
  const int bytes = dtype == PP_DTYPE_F32 ? 4 : 2;
  RotArgs a;
  a.x = x, a.y = y, a.pos = positions, a.inv_freq = inv_freq;
  for (int i = 0; i < 3; ++i) a.xs[i] = x_strides[i], a.ys[i] = y_strides[i];
  a.pb = pos_strides[0], a.pl = pos_strides[1];
  a.n = batch * length, a.L = (uint32_t)length, a.heads = (uint32_t)heads;
  a.D = D, a.rd = rotary_dim, a.pos64 = pos64, a.mscale = mscale, a.sign = inverse ? -1.0f : 1.0f;
  // 16-byte vectors where every head starts on one and the parts are whole vectors
  const bool vec = rotary_dim % 16 == 0 && D % 8 == 0 && rot_aligned(x, a.xs, 3, bytes) && rot_aligned(y, a.ys, 3, bytes);
  const int64_t units = (int64_t)heads * (vec ? rotary_dim / 16 + (D - rotary_dim) / 8 : rotary_dim / 2 + D - rotary_dim);
  // Enough tokens to keep a thread on four steps, as long as that leaves two workgroups for each CU;
  // a call smaller than that spreads every token's heads over workgroups of one step.
  const int64_t cus = pp_device_cus();
  const int64_t want = std::max<int64_t>(1, 4 * ROT_THREADS / units);
  a.tokens = (int)std::max<int64_t>(1, std::min<int64_t>({want, a.n / (2 * cus), ROT_TABLE / (rotary_dim / 2)}));
  const int64_t steps = (a.tokens * units + ROT_THREADS - 1) / ROT_THREADS;
  const int64_t gx = (a.n + a.tokens - 1) / a.tokens;
  const int64_t gy = std::max<int64_t>(1, std::min<int64_t>({steps, (2 * cus + gx - 1) / gx, 65535}));
  const dim3 grid((unsigned)gx, (unsigned)gy);
  hipStream_t st = (hipStream_t)stream;
#define ROT(T, V)                                                                            \
  do {                                                                                       \
    if (layout == PP_ROTARY_HALF) rotary_kernel<T, V, true><<<grid, ROT_THREADS, 0, st>>>(a); \
    else rotary_kernel<T, V, false><<<grid, ROT_THREADS, 0, st>>>(a);                        \
  } while (0)
  if (dtype == PP_DTYPE_F32) {
    if (vec) ROT(float, 8);
    else ROT(float, 1);
  } else {
    if (vec) ROT(bf16_t, 8);
    else ROT(bf16_t, 1);
  }
#undef ROT
  return pp_check_launch(what);
}

// ------------------------------------------------------------------ append
// A work item is 16 aligned positions of one sequence (so it lies in one page) and a block of heads
// of one kind: query, key or value. Sequence s has the items (start >> 4) + 2 s and on: n new tokens
// lie in at most (n >> 4) + 2 such groups. Query and key items turn their tokens' heads as above.
// The value pages keep a channel's tokens next to each other, so a value item reads 16 tokens of two
// channels per thread, a wave's lanes on consecutive channels, and writes them as two 16-byte vectors
// a channel; a group that is not full writes its tokens' elements one by one.
#define APP_THREADS 256
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
  int per, nqb, nkb;  // heads per block, blocks of query and of key heads
};

__device__ __forceinline__ uint32_t app_pair(const float* p) {
  const float2 f = *(const float2*)p;
  return f32_to_bf16x2(f.x, f.y);
}
__device__ __forceinline__ uint32_t app_pair(const bf16_t* p) { return *(const uint32_t*)p; }

template <typename T, int D, bool HALF>
__global__ __launch_bounds__(APP_THREADS) void kv_append_kernel(AppArgs a) {
  __shared__ float2 cs_s[APP_TOKENS * D / 2];
  const int tid = threadIdx.x;
  const int64_t t = blockIdx.x;
  const int s = paged_seq_of(a.seqs, t, [](int c, int s) { return (int64_t)(c >> 4) + 2 * s; });
  const int c0 = a.seqs.start(s), len = max(a.seqs.start(s + 1) - c0, 0);
  const bool tail = s == a.seqs.n_seqs;  // rows of no sequence
  const int64_t first = tail ? 0 : (int64_t)a.seqs.kv_lens[s] - len;
  const int64_t p0 = (first & ~(int64_t)(APP_TOKENS - 1)) + APP_TOKENS * (t - ((c0 >> 4) + 2 * s));
  const int lo = (int)max((int64_t)0, first - p0), hi = (int)min((int64_t)APP_TOKENS, first + len - p0);  // the group's tokens
  if (lo >= hi) return;
  const int row0 = c0 + (int)(p0 - first);  // row of the group's place 0
  const int kind = blockIdx.y < a.nqb ? 0 : blockIdx.y < a.nqb + a.nkb ? 1 : 2;
  const int h0 = (blockIdx.y - (kind == 0 ? 0 : kind == 1 ? a.nqb : a.nqb + a.nkb)) * a.per;
  const int nh = min(a.per, (kind == 0 ? a.Hq : a.Hkv) - h0), nt = hi - lo;
  if (tail) {
    if (kind == 0 && a.zero_tail)
      for (int k = tid; k < nt * nh * (D / 8); k += APP_THREADS) {
        const int i = k / (nh * (D / 8)), r = k - i * (nh * (D / 8));
        *(uint4*)(a.q_out + ((int64_t)(row0 + lo + i) * a.Hq + h0) * D + r * 8) = make_uint4(0, 0, 0, 0);
      }
    return;
  }
  const int ps = 1 << a.seqs.lp;
  int page = -1;
  if (kind != 0) {
    page = p0 < 0 ? -1 : a.seqs.page(a.seqs.entry(s, p0 >> a.seqs.lp));
    if (page < 0) return;
  }
  const int place = (int)(p0 & (ps - 1));
  if (kind == 2) {
    bf16_t* const to = a.v_pages + (((int64_t)page * a.Hkv + h0) * D << a.seqs.lp) + place;
    for (int k = tid; k < nh * (D / 2); k += APP_THREADS) {
      const int h = k / (D / 2), d = 2 * (k - h * (D / 2));
      const T* src = (const T*)a.v + (int64_t)row0 * a.vs[0] + (h0 + h) * a.vs[1] + d;
      uint32_t w[APP_TOKENS];
#pragma unroll
      for (int i = 0; i < APP_TOKENS; ++i) w[i] = i >= lo && i < hi ? app_pair(src + i * a.vs[0]) : 0u;
      bf16_t* dst = to + ((int64_t)(h * D + d) << a.seqs.lp);
      if (nt == APP_TOKENS) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t x = w[8 * g + 2 * i], y = w[8 * g + 2 * i + 1];
              o[i] = e ? (x >> 16) | (y & 0xffff0000u) : (x & 0xffffu) | (y << 16);
            }
            *(uint4*)(dst + ((int64_t)e << a.seqs.lp) + 8 * g) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < APP_TOKENS; ++i)
          if (i >= lo && i < hi) {
            dst[i] = (bf16_t)w[i];
            dst[i + ps] = (bf16_t)(w[i] >> 16);
          }
      }
    }
    return;
  }
  const int half = a.rd / 2;
  for (int k = tid; k < nt * half; k += APP_THREADS) {
    const int i = k / half;
    cs_s[k] = rot_entry(p0 + lo + i, a.inv_freq[k - i * half], a.mscale, 1.0f);
  }
  __syncthreads();
  const int nr = half / 8, per = nr + (D - a.rd) / 8, units = nh * per;
  const T* const x = (const T*)(kind == 0 ? a.q : a.k);
  const int64_t ts = kind == 0 ? a.qs[0] : a.ks[0], hs = kind == 0 ? a.qs[1] : a.ks[1];
  for (int k = tid; k < nt * units; k += APP_THREADS) {
    const int i = k / units, r = k - i * units, h = r / per, u = r - h * per;
    bf16_t* y = kind == 0 ? a.q_out + ((int64_t)(row0 + lo + i) * a.Hq + h0 + h) * D
                          : a.k_pages + ((((int64_t)page * a.Hkv + h0 + h) << a.seqs.lp) + place + lo + i) * D;
    rot_unit<T, bf16_t, 8, HALF>(x + (int64_t)(row0 + lo + i) * ts + (h0 + h) * hs, y, cs_s + i * half, u, nr, a.rd);
  }
}

int pp_paged_check(const char* what, int64_t n_tokens, int n_seqs, const void* cu_q, const void* kv_lens,
                   const void* block_table, int max_pages, const void* k_pages, const void* v_pages, int num_pages,
                   int page_size, int Hq, int Hkv, int D) {
  PP_REQUIRE(D == 64 || D == 128, PP_ERR_UNSUPPORTED, "%s: head size %d unsupported (64 or 128)", what, D);
  PP_REQUIRE(page_size >= 16 && page_size <= 4096 && paged_log2(page_size) >= 0, PP_ERR_UNSUPPORTED,
             "%s: page size %d unsupported (a power of two, 16 to 4096)", what, page_size);
  PP_REQUIRE(Hkv >= 1 && Hq >= 0 && Hq % Hkv == 0 && Hq <= 65536, PP_ERR_INVALID,
             "%s: %d query heads on %d key heads (need a multiple)", what, Hq, Hkv);
  PP_REQUIRE(n_seqs >= 0 && n_seqs <= (1 << 20) && max_pages >= 1 && num_pages >= 1, PP_ERR_INVALID,
             "%s: %d sequences, a table of %d pages, a cache of %d", what, n_seqs, max_pages, num_pages);
  PP_REQUIRE(n_tokens >= 0 && n_tokens * (int64_t)std::max(Hq, Hkv) <= 0x7fffffff, PP_ERR_UNSUPPORTED,
             "%s: %lld tokens of %d heads", what, (long long)n_tokens, std::max(Hq, Hkv));
  PP_REQUIRE((int64_t)max_pages * page_size <= (1 << 30), PP_ERR_UNSUPPORTED,
             "%s: a table of %d pages of %d tokens (at most 2^30 tokens)", what, max_pages, page_size);
  if (n_tokens == 0) return PP_OK;
  PP_REQUIRE(cu_q && k_pages && v_pages && (n_seqs == 0 || (kv_lens && block_table)), PP_ERR_INVALID,
             "%s: null pointer", what);
  PP_REQUIRE((((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0, PP_ERR_INVALID, "%s: pages not 16-byte aligned", what);
  return PP_OK;
}

extern "C" int pp_kv_append(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                            const void* v, const int64_t* v_strides, int dtype, int64_t n_tokens, int n_seqs,
                            const int32_t* cu_q, const int32_t* kv_lens, const int32_t* block_table, int max_pages,
                            int num_pages, int page_size, int Hq, int Hkv, int D, const double* inv_freq,
                            int rotary_dim, int layout, float mscale, void* k_pages, void* v_pages, void* q_out,
                            int zero_tail, void* stream) {
  const char* const what = "pp_kv_append";
  if (!q) Hq = 0;
  int rc = pp_paged_check(what, n_tokens, n_seqs, cu_q, kv_lens, block_table, max_pages, k_pages, v_pages, num_pages,
                          page_size, Hq, Hkv, D);
  if (rc) return rc;
  PP_REQUIRE(dtype == PP_DTYPE_F32 || dtype == PP_DTYPE_BF16, PP_ERR_INVALID, "%s: dtype %d", what, dtype);
  PP_REQUIRE(layout == PP_ROTARY_HALF || layout == PP_ROTARY_INTERLEAVED, PP_ERR_INVALID, "%s: layout %d", what, layout);
  if (!inv_freq) rotary_dim = 0;
  PP_REQUIRE(rotary_dim >= 0 && rotary_dim <= D && rotary_dim % 16 == 0, PP_ERR_UNSUPPORTED,
             "%s: rotary_dim %d unsupported (a multiple of 16 up to the head size %d)", what, rotary_dim, D);
  if (n_tokens == 0) return PP_OK;
  PP_REQUIRE(k && v && k_strides && v_strides && (!q || (q_strides && q_out)), PP_ERR_INVALID, "%s: null pointer", what);
  const int bytes = dtype == PP_DTYPE_F32 ? 4 : 2;
  PP_REQUIRE(rot_aligned(k, k_strides, 2, bytes) && rot_aligned(v, v_strides, 2, bytes) &&
                 (!q || (rot_aligned(q, q_strides, 2, bytes) && ((uintptr_t)q_out & 15) == 0)),
             PP_ERR_INVALID, "%s: every head of q, k, v and q_out must start on a 16-byte boundary", what);
  AppArgs a;
  a.seqs = {cu_q, kv_lens, block_table, (int)n_tokens, n_seqs, max_pages, num_pages, paged_log2(page_size)};
  a.q = q, a.k = k, a.v = v;
  for (int i = 0; i < 2; ++i) a.qs[i] = q ? q_strides[i] : 0, a.ks[i] = k_strides[i], a.vs[i] = v_strides[i];
  a.q_out = (bf16_t*)q_out, a.k_pages = (bf16_t*)k_pages, a.v_pages = (bf16_t*)v_pages;
  a.inv_freq = inv_freq, a.Hq = Hq, a.Hkv = Hkv, a.rd = rotary_dim, a.mscale = mscale, a.zero_tail = zero_tail;
  a.per = 4;
  a.nqb = (Hq + a.per - 1) / a.per, a.nkb = (Hkv + a.per - 1) / a.per;
  const dim3 grid((unsigned)((n_tokens >> 4) + 2 * ((int64_t)n_seqs + 1)), (unsigned)(a.nqb + 2 * a.nkb));
  hipStream_t st = (hipStream_t)stream;
#define APP(T, D_)                                                                                       \
  do {                                                                                                   \
    if (layout == PP_ROTARY_HALF) kv_append_kernel<T, D_, true><<<grid, APP_THREADS, 0, st>>>(a);        \
    else kv_append_kernel<T, D_, false><<<grid, APP_THREADS, 0, st>>>(a);                                \
  } while (0)
  if (dtype == PP_DTYPE_F32) {
    if (D == 64) APP(float, 64);
    else APP(float, 128);
  } else {
    if (D == 64) APP(bf16_t, 64);
    else APP(bf16_t, 128);
  }
#undef APP
  return pp_check_launch(what);
}
