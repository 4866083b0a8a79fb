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
// 2^-24 of the angle: 0.06 rad at a million radians. What float32 does not hold of that part, up to 2^-25 of a
// half turn, is added to cos and sin to first order (without it they were off by 9e-8, all of cos next to its
// zero).
//
// Memory bound: one read, one write. cos and sin of a workgroup's tokens are computed once into
// LDS, then its threads stream the tokens' heads in 16-byte vectors, the next step's loads ahead of the
// present one's stores. bf16, 8192 tokens of 36 heads of 128 (151 MB): 27.3 us, 5.5 TB/s, where a large
// copy reaches 5.05; float32, 16384 tokens of 12 heads (201 MB): 38.0 us, 5.3 TB/s; one token 2.2 us, a
// launch.
#include <algorithm>

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

struct RotArgs {
  const void* x;
  void* y;
  const void* pos;
  const double* inv_freq;
  int64_t xs[3], ys[3];  // strides of batch, token and head, in elements
  int64_t pb, pl;        // strides of the positions
  int64_t n;             // tokens
  uint32_t L;
  int heads, D, rd, pos64;
  float mscale, sign;
  int lgu, lgt, lgh;     // log2 of the threads on a head, of the tokens of a workgroup, of rd / 2 (rounded up)
};

template <typename T, int V, bool HALF>
__global__ __launch_bounds__(ROT_THREADS) void rotary_kernel(RotArgs a) {
  __shared__ float2 cs_s[ROT_TABLE];
  const int half = a.rd / 2, nr = half / V, per = nr + (a.D - a.rd) / V;
  const uint32_t n0 = blockIdx.x << a.lgt;
  const int nt = (int)min((uint32_t)1 << a.lgt, (uint32_t)a.n - n0);
  const RotLanes w(threadIdx.x, a.lgu, a.lgt);
  const uint32_t n = n0 + w.i, b = n / a.L, l = n - b * a.L;
  const T* const x = (const T*)a.x + b * a.xs[0] + l * a.xs[1];
  T* const y = (T*)a.y + b * a.ys[0] + l * a.ys[1];
  int h = w.h + w.hstep * blockIdx.y, u = w.u;
  bool more = w.i < nt && h < a.heads && u < per;
  RotUnit<T, V, HALF> now, next;
  if (more) now.load(x + h * a.xs[2], u, nr, a.rd);
  rot_table(cs_s, a.inv_freq, half, a.lgh, nt, a.mscale, a.sign, [&](int t) {
    const uint32_t n = n0 + t, b = n / a.L;
    const int64_t at = b * a.pb + (n - b * a.L) * a.pl;
    return a.pos64 ? ((const int64_t*)a.pos)[at] : (int64_t)((const int32_t*)a.pos)[at];
  });
  __syncthreads();
  while (more) {
    int h2 = h, u2 = u + (1 << a.lgu);
    if (u2 >= per) u2 = w.u, h2 += w.hstep * gridDim.y;
    more = h2 < a.heads;
    if (more) next.load(x + h2 * a.xs[2], u2, nr, a.rd);
    now.store(y + h * a.ys[2], cs_s + w.i * half, u, nr, a.rd);
    now = next, h = h2, u = u2;
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
  a.n = batch * length, a.L = (uint32_t)length, a.heads = heads;
  a.D = D, a.rd = rotary_dim, a.pos64 = pos64, a.mscale = mscale, a.sign = inverse ? -1.0f : 1.0f;
  // 16-byte vectors where every head starts on one and the parts are whole vectors. (float32 in steps of 8
  // pairs, whose two loads of a vector each meet every other 16 bytes: 16384 tokens of 12 heads 50 us.)
  const int V = 16 / bytes;
  const bool vec = rotary_dim % (2 * V) == 0 && D % V == 0 && rot_aligned(x, a.xs, 3, bytes) && rot_aligned(y, a.ys, 3, bytes);
  const int per = vec ? (rotary_dim / 2 + D - rotary_dim) / V : rotary_dim / 2 + D - rotary_dim;
  a.lgu = std::min(8, rot_log2up(per)), a.lgh = std::min(8, rot_log2up(rotary_dim / 2));
  // Enough tokens to keep a thread on four steps, as long as that leaves two workgroups for each CU;
  // a call smaller than that spreads every token's heads over workgroups of one step.
  const int64_t cus = pp_device_cus();
  a.lgt = 0;
  while (a.lgt < 4 && a.lgu + a.lgt < 8 && ((int64_t)heads * per << a.lgt) < 4 * ROT_THREADS &&
         (a.n >> (a.lgt + 1)) >= 2 * cus && ((rotary_dim / 2) << (a.lgt + 1)) <= ROT_TABLE)
    ++a.lgt;
  const int64_t gx = (a.n + (1 << a.lgt) - 1) >> a.lgt, hstep = (ROT_THREADS >> a.lgu) >> a.lgt;
  const int64_t gy = std::max<int64_t>(1, std::min<int64_t>((heads + hstep - 1) / hstep, (2 * cus + gx - 1) / gx));
  PP_REQUIRE(gx <= 0xffffff, PP_ERR_UNSUPPORTED, "%s: %lld tokens of this head size", what, (long long)a.n);
  const dim3 grid((unsigned)gx, (unsigned)gy);
  hipStream_t st = (hipStream_t)stream;
#define ROT(T, V)                                                                            \
  do {                                                                                       \
    if (layout == PP_ROTARY_HALF) rotary_kernel<T, V, true><<<grid, ROT_THREADS, 0, st>>>(a); \
    else rotary_kernel<T, V, false><<<grid, ROT_THREADS, 0, st>>>(a);                        \
  } while (0)
  if (dtype == PP_DTYPE_F32) {
    if (vec) ROT(float, 4);
    else ROT(float, 1);
  } else {
    if (vec) ROT(bf16_t, 8);
    else ROT(bf16_t, 1);
  }
#undef ROT
  return pp_check_launch(what);
}

// ------------------------------------------------------------------ append
// A work item is a group of 16 aligned positions of one sequence (so it lies in one page) and a block
// of query or of key heads, or four such groups and a block of value heads. Sequence s has the items
// (start >> 4) + 2 s and on: n new tokens lie in at most (n >> 4) + 2 groups (and 6 for 4 of the value
// items). Query and key items turn their tokens' heads as above. The value pages keep a channel's
// tokens next to each other: a thread reads 16 tokens of two channels, a wave's lanes on consecutive
// channels, and writes them as two 16-byte vectors a channel; a group that is not full writes its
// tokens' elements one by one. The waves of a value item take its four groups, so that in pages of 64
// and more the 128 bytes of a channel leave the same L2 together.
// Bound by memory for chunks (8192 tokens of 36 heads, 151 MB: 37 us, 4.1 TB/s; the rotation alone of as
// many bytes 27.3), by the chain offsets, table, rows for single tokens (3.9 us for one, 5.4 for 64, 9.1
// for 256 of them).
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

__device__ __forceinline__ uint32_t app_pair(const float* p) {
  const float2 f = *(const float2*)p;
  return f32_to_bf16x2(f.x, f.y);
}
__device__ __forceinline__ uint32_t app_pair(const bf16_t* p) { return *(const uint32_t*)p; }

template <typename T, int D, bool HALF>
__global__ __launch_bounds__(APP_THREADS) void kv_append_kernel(AppArgs a) {
  __shared__ float2 cs_s[APP_TOKENS * D / 2];
  const int tid = threadIdx.x;
  // the grid: value items, whose way is the longest, then query and key items
  const bool value = blockIdx.x < a.values;
  const uint32_t id = value ? blockIdx.x : blockIdx.x - a.values, nb = value ? a.nvb : a.nqb + a.nkb;
  const uint32_t block = id % nb, t = id / nb;
  const int kind = value ? 2 : block < (uint32_t)a.nqb ? 0 : 1;
  const int h0 = value ? block * a.vper : (block - (kind ? a.nqb : 0)) * a.per;
  const int nh = min(value ? a.vper : a.per, (kind ? a.Hkv : a.Hq) - h0);
  const int lg = value ? 6 : 4;  // log2 of the item's positions
  // what does not depend on the sequence is asked for before it is found, and further down the table's entry
  // before the rows: the chain of loads is what a call of single tokens takes
  const int half = a.rd / 2, pair = tid & ((1 << a.lgh) - 1);
  const double freq = half ? a.inv_freq[min(pair, half - 1)] : 0.0;
  const PagedSeq f = paged_find(a.seqs, t, [lg](int c, int s) { return (int64_t)(c >> lg) + 2 * s; });
  const int s = f.s, c0 = f.c0, len = f.rows;
  const bool tail = s == a.seqs.n_seqs;  // rows of no sequence
  const int64_t first = tail ? 0 : (int64_t)f.len - len;
  int64_t p0 = ((first >> lg) + (t - ((c0 >> lg) + 2 * s))) << lg;
  // value items: their four groups to the four waves, unless only one has tokens
  bool alone = true;
  if (value) {
    const int64_t from = max(p0, first & ~(int64_t)(APP_TOKENS - 1));
    alone = min(p0 + 64, first + len) - from <= APP_TOKENS;
    p0 = alone ? from : p0 + APP_TOKENS * __builtin_amdgcn_readfirstlane(tid >> 6);
  }
  const int lo = (int)max((int64_t)0, first - p0), hi = (int)min((int64_t)APP_TOKENS, first + len - p0);  // the group's tokens
  if (lo >= hi) return;
  const int row0 = c0 + (int)(p0 - first);  // row of the group's place 0
  const int nt = hi - lo;
  if (tail) {
    if (kind == 0 && a.zero_tail)
      for (int k = tid; k < nt * nh * (D / 8); k += APP_THREADS) {
        const int i = k / (nh * (D / 8)), r = k - i * (nh * (D / 8));
        *(uint4*)(a.q_out + ((int64_t)(row0 + lo + i) * a.Hq + h0) * D + r * 8) = make_uint4(0, 0, 0, 0);
      }
    return;
  }
  const int ps = 1 << a.seqs.lp;
  const int64_t at = p0 >> a.seqs.lp;
  const int entry = kind ? a.seqs.table[(int64_t)s * a.seqs.max_pages + min(max(at, (int64_t)0), (int64_t)a.seqs.max_pages - 1)] : 0;
  paged_asked();
  const bool place_ok = at >= 0 && at < a.seqs.max_pages;
  auto no_page = [&] { return !place_ok || a.seqs.page(entry) < 0; };
  const int place = (int)(p0 & (ps - 1));
  if (kind == 2) {
    constexpr int P = D / 2;  // pairs of channels of a head
    bf16_t* const to = a.v_pages + (((int64_t)entry * a.Hkv + h0) * D << a.seqs.lp) + place;
    for (int k = alone ? tid : tid & 63; k < nh * P; k += alone ? APP_THREADS : 64) {
      const int h = k / P, d = 2 * (k - h * P);
      const T* src = (const T*)a.v + (int64_t)row0 * a.vs[0] + (h0 + h) * a.vs[1] + d;
      bf16_t* dst = to + ((int64_t)(h * D + d) << a.seqs.lp);
      if (nt == APP_TOKENS) {
        uint32_t w[APP_TOKENS];
#pragma unroll
        for (int i = 0; i < APP_TOKENS; ++i) w[i] = app_pair(src + i * a.vs[0]);
        paged_asked();
        if (no_page()) return;
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
        uint32_t w = app_pair(src + lo * a.vs[0]);
        paged_asked();
        if (no_page()) return;
        dst[lo] = (bf16_t)w;
        dst[lo + ps] = (bf16_t)(w >> 16);
#pragma unroll 4
        for (int i = lo + 1; i < hi; ++i) {
          w = app_pair(src + i * a.vs[0]);
          dst[i] = (bf16_t)w;
          dst[i + ps] = (bf16_t)(w >> 16);
        }
      }
    }
    return;
  }
  const int nr = half / 8, per = nr + (D - a.rd) / 8;
  const RotLanes w(tid, a.lgu, 32 - __clz(nt - 1));  // as many tokens as there are
  const int64_t row = row0 + lo + w.i;
  const T* const x = (const T*)(kind == 0 ? a.q : a.k) + row * (kind == 0 ? a.qs[0] : a.ks[0]);
  const int64_t xs = kind == 0 ? a.qs[1] : a.ks[1];
  bf16_t* const y = kind == 0 ? a.q_out + row * a.Hq * D
                              : a.k_pages + (((int64_t)entry * a.Hkv << a.seqs.lp) + place + lo + w.i) * D;
  const int64_t ys = kind == 0 ? D : (int64_t)D << a.seqs.lp;
  int h = h0 + w.h;
  bool more = w.i < nt && h < h0 + nh && w.u < per;
  RotUnit<T, 8, HALF> now, next;
  if (more) now.load(x + h * xs, w.u, nr, a.rd);
  paged_asked();
  if (pair < half)
    for (int t = tid >> a.lgh; t < nt; t += APP_THREADS >> a.lgh) cs_s[t * half + pair] = rot_entry(p0 + lo + t, freq, a.mscale, 1.0f);
  if (kind && no_page()) return;
  __syncthreads();
  while (more) {
    const int h2 = h + w.hstep;
    more = h2 < h0 + nh;
    if (more) next.load(x + h2 * xs, w.u, nr, a.rd);
    now.store(y + h * ys, cs_s + w.i * half, w.u, nr, a.rd);
    now = next, h = h2;
  }
}

int pp_paged_sizes(const char* what, int64_t n_tokens, int n_seqs, int max_pages, int num_pages, int page_size, int Hq,
                   int Hkv, int D) {
  PP_REQUIRE(D == 64 || D == 128, PP_ERR_UNSUPPORTED, "%s: head size %d unsupported (64 or 128)", what, D);
  PP_REQUIRE(page_size >= 16 && page_size <= 4096 && paged_log2(page_size) >= 0, PP_ERR_UNSUPPORTED,
             "%s: page size %d unsupported (a power of two, 16 to 4096)", what, page_size);
  PP_REQUIRE(Hkv >= 1 && Hq >= 0 && Hq % Hkv == 0 && Hq <= 65536, PP_ERR_INVALID,
             "%s: %d query heads on %d key heads (need a multiple)", what, Hq, Hkv);
  PP_REQUIRE(n_seqs >= 0 && n_seqs <= (1 << 20) && max_pages >= 1 && num_pages >= 1, PP_ERR_INVALID,
             "%s: %d sequences, a table of %d pages, a cache of %d", what, n_seqs, max_pages, num_pages);
  PP_REQUIRE(n_tokens >= 0 && n_tokens <= 0x7fffffff / std::max(Hq, Hkv), PP_ERR_UNSUPPORTED,
             "%s: %lld tokens of %d heads", what, (long long)n_tokens, std::max(Hq, Hkv));
  PP_REQUIRE((int64_t)max_pages * page_size <= (1 << 30), PP_ERR_UNSUPPORTED,
             "%s: a table of %d pages of %d tokens (at most 2^30 tokens)", what, max_pages, page_size);
  return PP_OK;
}

int pp_paged_check(const char* what, int64_t n_tokens, int n_seqs, const void* cu_q, const void* kv_lens,
                   const void* block_table, int max_pages, const void* k_pages, const void* v_pages, int num_pages,
                   int page_size, int Hq, int Hkv, int D) {
  const int rc = pp_paged_sizes(what, n_tokens, n_seqs, max_pages, num_pages, page_size, Hq, Hkv, D);
  if (rc || n_tokens == 0) return rc;
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
  a.lgu = rot_log2up(rotary_dim / 16 + (D - rotary_dim) / 8), a.lgh = rot_log2up(std::max(rotary_dim / 2, 1));
  // Heads of an item. Single tokens: a group has one, so all the heads that the threads hold in one step
  // (32, value heads 4, or 16 where there are workgroups enough); 1, 64, 256 sequences of 12 heads 3.5,
  // 5.1, 8.8 us, in items of 4 heads 3.7, 5.7, 12.6. Chunks: 4, and one value head (64 tokens of it),
  // 8192 tokens (151 MB, from memory) 38 us, 8 or 12 heads 42 and 41. Between them, and where a chunk is among
  // single tokens, 4 value heads: 64 sequences of 4 and 16 tokens 8.7 and 16.6 us, with 16 13.4 and 27.5; 64
  // single tokens and 512 8.9 against 13.2, 255 and 3800 24 against 34 (with one 31).
  a.per = n_tokens <= 4 * (int64_t)n_seqs ? 32 : 4;
  a.vper = n_tokens > 16 * (int64_t)n_seqs ? 1 : n_seqs >= 64 && n_tokens <= 2 * (int64_t)n_seqs ? 16 : 4;
  a.nqb = (Hq + a.per - 1) / a.per, a.nkb = (Hkv + a.per - 1) / a.per, a.nvb = (Hkv + a.vper - 1) / a.vper;
  const int64_t values = ((n_tokens >> 6) + 2 * ((int64_t)n_seqs + 1)) * a.nvb;
  const int64_t items = values + ((n_tokens >> 4) + 2 * ((int64_t)n_seqs + 1)) * (a.nqb + a.nkb);
  PP_REQUIRE(items <= 0xffffff, PP_ERR_UNSUPPORTED, "%s: %lld work items (at most 2^24 - 1)", what, (long long)items);
  a.values = (uint32_t)values;
  const unsigned grid = (unsigned)items;
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
