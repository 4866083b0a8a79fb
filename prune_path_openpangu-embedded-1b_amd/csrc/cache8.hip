// The append to a paged cache of 8 bits, and the read of a paged cache of either kind back to packed rows.
//
// Keys [page][head][place][channel] as in the cache of 16 bits; values [page][head][block of 16 places][channel][16]: a
// channel's 16 tokens, one 16-byte word, are what an append transposes and what a lane of the attention takes, and a
// block is 16 D contiguous bytes whatever the page size. Scales [page][head][block].
//
// A wave takes one block of one head (at D = 64 two heads of values): its values' largest magnitude is a fold over the
// wave, and the block has no other writer, so old tokens are brought to a larger scale in place. The scale of a block
// is the least that holds its values; where the block held tokens before (places in front of the call's first
// token in it), at least the one that it had.
//
// Memory bound for chunks: 8192 tokens of 12 query, key and value heads (126 MB) 29.0 us, with the norms 31.6 (4.0 TB/s; 95
// registers, five waves a SIMD: fewer spill, and four channels a lane instead of two, for wider loads of V, 38 us); half of the
// channels turned 38.9 (145 registers, three waves). The chain offsets, table, rows and scale for single tokens: 4.5 us for one,
// 5.1 for 32 of them, 12.3 for 256 (with norms 4.8, 5.3, 12.7). The read: 64 sequences of 12 heads, 2.26 GB, 453 us (5.0 TB/s,
// a large copy's rate).
#include <algorithm>

#include "append.h"
#include "fp8.h"

__device__ __forceinline__ uint32_t c8_max(uint32_t a, uint32_t b) { return max(a, b); }
__device__ __forceinline__ uint32_t c8_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// The largest of LANES neighbours, a power of two from 32 on.
template <int LANES>
__device__ __forceinline__ uint32_t c8_fold(uint32_t v) {
  const int lane = threadIdx.x & 63;
  auto of = [](float f) { return __float_as_uint(f); };
  v = c8_max(v, of(dpp_mov<PP_DPP_ROR8>(__uint_as_float(v))));
  v = c8_max(v, of(dpp_mov<PP_DPP_ROR4>(__uint_as_float(v))));
  v = c8_max(v, of(dpp_mov<PP_DPP_XOR2>(__uint_as_float(v))));
  v = c8_max(v, of(dpp_mov<PP_DPP_XOR1>(__uint_as_float(v))));
  v = c8_max(v, pl_xor16(v, lane));
  if (LANES == 64) v = c8_max(v, pl_xor32(v, lane));
  return v;
}

__device__ __forceinline__ float2 c8_pair(const float* p) { return *(const float2*)p; }
__device__ __forceinline__ float2 c8_pair(const bf16_t* p) {
  const uint32_t w = *(const uint32_t*)p;
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// The finite ones of N magnitudes' largest, of all LANES lanes, if any lane has one that is not below FP8_TOP.
template <int LANES, int N>
__device__ __forceinline__ uint32_t c8_top(const float (&x)[N], bool& odd) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) top = c8_max(top, c8_bits(x[i]));
  top = c8_fold<LANES>(top);
  odd = __ballot(top > FP8_TOP) != 0;
  if (__builtin_expect(odd, 0)) {
    top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) top = c8_max(top, c8_bits(x[i]) < 0x7f800000u ? c8_bits(x[i]) : 0u);
    top = c8_fold<LANES>(top);
  }
  return top;
}

#define C8_FEW 4  // new tokens of a block up to which its values go out byte by byte

// x * inv as the cache takes it; `odd`: some value of the wave is not finite or beyond the largest scale's 448.
template <int N>
__device__ __forceinline__ void c8_scale(float (&x)[N], float inv, bool odd) {
  if (__builtin_expect(odd, 0)) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = fp8_odd(x[i], inv);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= inv;
  }
}

template <typename T, int D, bool HALF, bool FULL>
__global__ __launch_bounds__(APP_THREADS) void kv_append8_kernel(AppArgs a, AppMore more) {
  constexpr int LGU = (D == 64 ? 2 : 3) + !FULL, SLOTS = 64 >> LGU, NP = APP_TOKENS / SLOTS;  // key items
  constexpr int P = D / 2, HW = 64 / P;                                                       // value items: lanes of a head, heads of a wave
  __shared__ float2 cs_s[APP_TOKENS * D / 2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool value = blockIdx.x < a.values;
  const uint32_t id = value ? blockIdx.x : blockIdx.x - a.values, nb = value ? a.nvb : a.nqb + a.nkb;
  const uint32_t block = id % nb, t = id / nb;
  const int kind = value ? 2 : block < (uint32_t)a.nqb ? 0 : 1;
  // what does not depend on the sequence is asked for before it is found, and the table's entry before the rows
  const int half = a.rd / 2, pair = tid & ((1 << a.lgh) - 1);
  const double freq = half && !value ? a.inv_freq[min(pair, half - 1)] : 0.0;
  const PagedSeq f = paged_find(a.seqs, t, [](int c, int s) { return (int64_t)(c >> 4) + 2 * s; });
  const int s = f.s, c0 = f.c0, len = f.rows;
  const bool tail = s == a.seqs.n_seqs;  // rows of no sequence
  const int64_t first = tail ? 0 : (int64_t)f.len - len;
  const int64_t p0 = ((first >> 4) + (t - ((c0 >> 4) + 2 * s))) << 4;
  const int lo = (int)max((int64_t)0, first - p0), hi = (int)min((int64_t)APP_TOKENS, first + len - p0);  // the block's new tokens
  if (lo >= hi) return;
  const int nt = hi - lo;
  const int64_t row0 = c0 + (p0 - first) + lo;  // the first of them
  if (tail) {
    const int h0 = block * a.per, nh = min(a.per, a.Hq - h0);
    if (kind == 0 && a.zero_tail)
      for (int k = tid; k < nt * nh * (D / 8); k += APP_THREADS) {
        const int i = k / (nh * (D / 8)), r = k - i * (nh * (D / 8));
        *(uint4*)(a.q_out + ((row0 + i) * a.Hq + h0) * D + r * 8) = make_uint4(0, 0, 0, 0);
      }
    return;
  }
  if (kind == 0) {
    const int h0 = block * a.per;
    auto drop = [] { return false; };
    bf16_t* const to = a.q_out + row0 * a.Hq * D;
    if (more.qw) app_turn<T, D, HALF, true>(a, more, 0, cs_s, freq, pair, half, row0, nt, h0, min(a.per, a.Hq - h0), p0 + lo, to, (int64_t)a.Hq * D, D, drop);
    else app_turn<T, D, HALF, false>(a, more, 0, cs_s, freq, pair, half, row0, nt, h0, min(a.per, a.Hq - h0), p0 + lo, to, (int64_t)a.Hq * D, D, drop);
    return;
  }
  const int64_t at = p0 >> a.seqs.lp;
  const bool place_ok = at >= 0 && at < a.seqs.max_pages;
  const int entry = a.seqs.table[(int64_t)s * a.seqs.max_pages + min(max(at, (int64_t)0), (int64_t)a.seqs.max_pages - 1)];
  paged_asked();
  const int place = (int)(p0 & ((1 << a.seqs.lp) - 1)), lb = a.seqs.lp - 4;
  if (value) {
    const int h = (block * 4 + wave) * HW + lane / P, l = lane % P;  // channels 2 l and 2 l + 1
    const bool on = h < a.Hkv;
    const T* const src = (const T*)a.v + row0 * a.vs[0] + (on ? h : 0) * a.vs[1] + 2 * l;
    auto where = [&](int page) { return (((int64_t)page * a.Hkv + (on ? h : 0)) << lb) + (place >> 4); };
    // A few tokens go out byte by byte, unless older ones change, and skip what the places of a whole block take
    // (256 single tokens of 12 heads 12.3 us, as a block's whole words 13.7; 32 5.1 and 5.5).
    if (nt <= C8_FEW) {
      float x[2 * C8_FEW];
#pragma unroll
      for (int i = 0; i < C8_FEW; ++i) {
        const float2 w = c8_pair(src + min(i, nt - 1) * a.vs[0]);
        x[2 * i] = on && i < nt ? w.x : 0.0f, x[2 * i + 1] = on && i < nt ? w.y : 0.0f;
      }
      paged_asked();
      const int page = place_ok ? a.seqs.page(entry) : -1;
      if (page < 0) return;
      const int64_t to = where(page);
      const int held = lo > 0 ? more.v_scales[to] : FP8_LOW;
      bool odd;
      const int byte = max(fp8_scale(c8_top<P>(x, odd)), min(max(held, FP8_LOW), FP8_HIGH));
      if (__ballot(lo > 0 && byte != held) == 0) {
        const float inv = fp8_inverse(byte);
        c8_scale(x, inv, odd);
        uint8_t* const dst = more.v8 + to * (APP_TOKENS * D) + 32 * l + lo;
#pragma unroll
        for (int i = 0; i < C8_FEW; ++i)
          if (on && i < nt) {
            const uint32_t w = fp8_pack(x[2 * i], x[2 * i + 1], 0.0f, 0.0f);
            dst[i] = (uint8_t)w, dst[i + 16] = (uint8_t)(w >> 8);
          }
        if (on && l == 0 && lo == 0) more.v_scales[to] = (uint8_t)byte;
        return;
      }
    }
    float x[2 * APP_TOKENS];
#pragma unroll
    for (int i = 0; i < APP_TOKENS; ++i) {
      const float2 w = c8_pair(src + min(max(i - lo, 0), nt - 1) * a.vs[0]);
      x[i] = on && i >= lo && i < hi ? w.x : 0.0f;
      x[APP_TOKENS + i] = on && i >= lo && i < hi ? w.y : 0.0f;
    }
    paged_asked();
    const int page = place_ok ? a.seqs.page(entry) : -1;
    if (page < 0) return;
    const int64_t to = where(page);
    uint4* const dst = (uint4*)(more.v8 + to * (APP_TOKENS * D)) + 2 * l;
    uint8_t* const scale = more.v_scales + to;
    uint4 was[2] = {};
    const int held = lo > 0 ? *scale : FP8_LOW;
    if (nt < APP_TOKENS) was[0] = dst[0], was[1] = dst[1];  // the other places' bytes stay
    bool odd;
    const int byte = max(fp8_scale(c8_top<P>(x, odd)), min(max(held, FP8_LOW), FP8_HIGH));
    const float inv = fp8_inverse(byte), bring = fp8_step(held, byte);
    c8_scale(x, inv, odd);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float* const v = x + APP_TOKENS * e + 4 * j;
        w[j] = fp8_pack(v[0], v[1], v[2], v[3]);
      }
      if (nt < APP_TOKENS) {
        const uint32_t before[4] = {was[e].x, was[e].y, was[e].z, was[e].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t fresh = 0, kept = 0;  // the new tokens' bytes, and those before them
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            fresh |= 4 * j + i >= lo && 4 * j + i < hi ? 0xffu << (8 * i) : 0u;
            kept |= 4 * j + i < lo ? 0xffu << (8 * i) : 0u;
          }
          const uint32_t old = lo > 0 && byte != held ? (fp8_rescale(before[j], bring) & kept) | (before[j] & ~kept) : before[j];
          w[j] = (w[j] & fresh) | (old & ~fresh);
        }
      }
      if (on) dst[e] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (on && l == 0) *scale = (uint8_t)byte;
    return;
  }
  // keys
  const int u = lane & ((1 << LGU) - 1), slot = lane >> LGU;
  const int h = (block - a.nqb) * 4 + wave;
  const bool on = h < a.Hkv;
  const int nr = half / 8, per = nr + (D - a.rd) / 8;
  RotUnit<T, 8, HALF> x[NP];
  const T* const src = (const T*)a.k + row0 * a.ks[0] + (on ? h : 0) * a.ks[1];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    if (i * SLOTS >= nt) break;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[i].p.v[j] = x[i].q.v[j] = 0;
    const int n = i * SLOTS + slot;
    if (on && n < nt && u < per) x[i].load(src + n * a.ks[0], u, nr, a.rd);
  }
  float wa[8], wb[8];
  if (more.kw) rot_weights<8, HALF>(more.kw, more.w32, u, nr, per, a.rd, wa, wb);
  paged_asked();
  if (pair < half)
    for (int n = tid >> a.lgh; n < nt; n += APP_THREADS >> a.lgh) cs_s[n * half + pair] = rot_entry(p0 + lo + n, freq, a.mscale, 1.0f);
  const int page = place_ok ? a.seqs.page(entry) : -1;
  if (page < 0) return;
  const int64_t to = (((int64_t)page * a.Hkv + (on ? h : 0)) << lb) + (place >> 4);
  const int held = lo > 0 ? more.k_scales[to] : FP8_LOW;
  paged_asked();
  __syncthreads();
  if (!on) return;  // the whole wave
  uint8_t* const dst = more.k8 + to * (APP_TOKENS * D);
  float y[2 * 8 * NP];
#pragma unroll
  for (int i = 0; i < 2 * 8 * NP; ++i) y[i] = 0.0f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    if (i * SLOTS >= nt) break;
    float p[8], q[8];
    rot_pairs(x[i], u < nr, p, q);
    if (more.kw) app_norm<T, HALF>(wa, wb, D, more.eps, LGU, p, q);
    const int n = i * SLOTS + slot;
    const bool mine = n < nt && u < per;
    if (mine && u < nr) rot_turn<8>(cs_s + n * half + u * 8, p, q);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[16 * i + j] = mine ? p[j] : 0.0f, y[16 * i + 8 + j] = mine ? q[j] : 0.0f;
  }
  bool odd;
  const int byte = max(fp8_scale(c8_top<64>(y, odd)), min(max(held, FP8_LOW), FP8_HIGH));
  const float inv = fp8_inverse(byte);
  if (lo > 0 && byte != held) {  // (a block of elsewhere may have any scale)
    const float bring = fp8_step(held, byte);
    for (int c = lane; c < lo * (D / 16); c += 64) {
      const uint4 w = ((const uint4*)dst)[c];
      ((uint4*)dst)[c] = make_uint4(fp8_rescale(w.x, bring), fp8_rescale(w.y, bring), fp8_rescale(w.z, bring), fp8_rescale(w.w, bring));
    }
  }
  c8_scale(y, inv, odd);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    if (i * SLOTS >= nt) break;
    const float* const v = y + 16 * i;
    const int n = i * SLOTS + slot;
    if (n >= nt || u >= per) continue;
    uint8_t* const row = dst + (lo + n) * D;
    if (u >= nr) {
      *(uint2*)(row + a.rd + 8 * (u - nr)) = make_uint2(fp8_pack(v[0], v[1], v[2], v[3]), fp8_pack(v[4], v[5], v[6], v[7]));
    } else if (HALF) {
      *(uint2*)(row + 8 * u) = make_uint2(fp8_pack(v[0], v[1], v[2], v[3]), fp8_pack(v[4], v[5], v[6], v[7]));
      *(uint2*)(row + a.rd / 2 + 8 * u) = make_uint2(fp8_pack(v[8], v[9], v[10], v[11]), fp8_pack(v[12], v[13], v[14], v[15]));
    } else {
      *(uint4*)(row + 16 * u) = make_uint4(fp8_pack(v[0], v[8], v[1], v[9]), fp8_pack(v[2], v[10], v[3], v[11]),
                                           fp8_pack(v[4], v[12], v[5], v[13]), fp8_pack(v[6], v[14], v[7], v[15]));
    }
  }
  if (lane == 0) more.k_scales[to] = (uint8_t)byte;
}

int app8_launch(const char* what, AppArgs& a, const AppMore& e, int dtype, int D, int layout, int64_t n_tokens, hipStream_t st) {
  const int vheads = 512 / D;
  // Query heads of an item: as of the 16-bit cache for single tokens; 8 for chunks. us for 4, 8, 12 heads, 8192 tokens: 12 query and key
  // heads 30.1, 29.7, 36.7 (with norms 30.2, 31.0, 38.3), 16 36.9, 34.4, 39.6 (38.1, 37.2, 42.3), 32 81, 74, 75; 20 on 4 23.3, 23.9, 23.9;
  // 4 chunks of 2048, 24 on 8, 31.6, 29.8, 34.3 (33.4, 31.7, 36.5).
  a.per = n_tokens <= 4 * (int64_t)a.seqs.n_seqs ? 32 : 8;
  a.nqb = (a.Hq + a.per - 1) / a.per, a.nkb = (a.Hkv + 3) / 4, a.nvb = (a.Hkv + vheads - 1) / vheads;
  const int64_t groups = (n_tokens >> 4) + 2 * ((int64_t)a.seqs.n_seqs + 1), items = groups * (a.nqb + a.nkb + a.nvb);
  PP_REQUIRE(items <= 0xffffff, PP_ERR_UNSUPPORTED, "%s: %lld work items (at most 2^24 - 1)", what, (long long)items);
  a.values = (uint32_t)(groups * a.nvb);
  const unsigned grid = (unsigned)items;
#define APP8_FULL(T, D_, HALF_)                                                                        \
  do {                                                                                                 \
    if (a.rd == D_) kv_append8_kernel<T, D_, HALF_, true><<<grid, APP_THREADS, 0, st>>>(a, e);         \
    else kv_append8_kernel<T, D_, HALF_, false><<<grid, APP_THREADS, 0, st>>>(a, e);                   \
  } while (0)
#define APP8(T, D_)                                             \
  do {                                                          \
    if (layout == PP_ROTARY_HALF) APP8_FULL(T, D_, true);       \
    else APP8_FULL(T, D_, false);                               \
  } while (0)
  if (dtype == PP_DTYPE_F32) {
    if (D == 64) APP8(float, 64);
    else APP8(float, 128);
  } else {
    if (D == 64) APP8(bf16_t, 64);
    else APP8(bf16_t, 128);
  }
#undef APP8
#undef APP8_FULL
  return pp_check_launch(what);
}

// ------------------------------------------------------------------ read
// A wave takes 16 places of one head (at D = 64 two heads of values), as above; the rows go out as the batch
// lies, [row][head][channel]. Rows whose place no page holds are zeros.
struct ReadArgs {
  PagedSeqs seqs;
  const void *k, *v;
  const uint8_t *k_scales, *v_scales;
  bf16_t *k_out, *v_out;
  int Hkv, zero_tail;
  int nkb, nvb;  // workgroups to the key heads and to the value heads of 16 places
};

template <int D, bool EIGHT>
__global__ __launch_bounds__(APP_THREADS) void kv_read_kernel(ReadArgs a) {
  constexpr int P = D / 2, HW = 64 / P;  // lanes of a value head, value heads of a wave
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t nb = a.nkb + a.nvb, block = blockIdx.x % nb, t = blockIdx.x / nb;
  const bool value = block >= (uint32_t)a.nkb;
  const PagedSeq f = paged_find(a.seqs, t, [](int c, int s) { return (int64_t)(c >> 4) + 2 * s; });
  const int s = f.s, c0 = f.c0, len = f.rows;
  const bool tail = s == a.seqs.n_seqs;
  const int64_t first = tail ? 0 : (int64_t)f.len - len;
  const int64_t p0 = ((first >> 4) + (t - ((c0 >> 4) + 2 * s))) << 4;
  const int lo = (int)max((int64_t)0, first - p0), hi = (int)min((int64_t)APP_TOKENS, first + len - p0);
  if (lo >= hi || (tail && !a.zero_tail)) return;
  const int64_t row0 = c0 + (p0 - first);  // row of place 0
  const int64_t at = p0 >> a.seqs.lp;
  int page = -1;
  if (!tail && at >= 0 && at < a.seqs.max_pages) page = a.seqs.page(a.seqs.table[(int64_t)s * a.seqs.max_pages + at]);
  const int place = (int)(p0 & ((1 << a.seqs.lp) - 1)), lb = a.seqs.lp - 4;
  if (value) {
    const int h = ((block - a.nkb) * 4 + wave) * HW + lane / P, l = lane % P;  // channels 2 l and 2 l + 1
    if (h >= a.Hkv) return;
    uint32_t x[2][8];  // of each channel the 16 tokens, in pairs
    if (page < 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[0][i] = x[1][i] = 0;
    } else if (EIGHT) {
      const int64_t from = (((int64_t)page * a.Hkv + h) << lb) + (place >> 4);
      const uint4* const src = (const uint4*)((const uint8_t*)a.v + from * (APP_TOKENS * D)) + 2 * l;
      const float scale = fp8_factor(a.v_scales[from]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 w = src[e];
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[e][2 * i] = fp8_bf16<false>(v[i], scale), x[e][2 * i + 1] = fp8_bf16<true>(v[i], scale);
      }
    } else {
      const bf16_t* const src = (const bf16_t*)a.v + ((((int64_t)page * a.Hkv + h) * D + 2 * l) << a.seqs.lp) + place;
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 w = *(const uint4*)(src + ((int64_t)e << a.seqs.lp) + 8 * i);
          x[e][4 * i] = w.x, x[e][4 * i + 1] = w.y, x[e][4 * i + 2] = w.z, x[e][4 * i + 3] = w.w;
        }
    }
    bf16_t* const dst = a.v_out + (row0 * a.Hkv + h) * D + 2 * l;
#pragma unroll
    for (int i = 0; i < APP_TOKENS; ++i) {
      const uint32_t u = x[0][i / 2], v = x[1][i / 2];
      if (i >= lo && i < hi)
        *(uint32_t*)(dst + (int64_t)i * a.Hkv * D) = i & 1 ? (u >> 16) | (v & 0xffff0000u) : (u & 0xffffu) | (v << 16);
    }
    return;
  }
  const int h = block * 4 + wave;
  if (h >= a.Hkv) return;
  const int64_t from = ((((int64_t)max(page, 0) * a.Hkv + h) << lb) + (place >> 4));
  bf16_t* const dst = a.k_out + (row0 * a.Hkv + h) * D;
  constexpr int C = D / 16;  // pieces of 16 channels
#pragma unroll
  for (int i = 0; i < APP_TOKENS * C / 64; ++i) {
    const int c = 64 * i + lane, n = c / C, d = c % C * 16;
    uint4 o[2] = {};
    if (page >= 0 && n >= lo && n < hi) {
      if (EIGHT) {
        const float scale = fp8_factor(a.k_scales[from]);
        const uint4 w = ((const uint4*)((const uint8_t*)a.k + from * (APP_TOKENS * D)))[c];
        o[0] = make_uint4(fp8_bf16<false>(w.x, scale), fp8_bf16<true>(w.x, scale), fp8_bf16<false>(w.y, scale), fp8_bf16<true>(w.y, scale));
        o[1] = make_uint4(fp8_bf16<false>(w.z, scale), fp8_bf16<true>(w.z, scale), fp8_bf16<false>(w.w, scale), fp8_bf16<true>(w.w, scale));
      } else {
        const uint4* const src = (const uint4*)((const bf16_t*)a.k + from * (APP_TOKENS * D)) + 2 * c;
        o[0] = src[0], o[1] = src[1];
      }
    }
    if (n >= lo && n < hi) {
      uint4* const to = (uint4*)(dst + (int64_t)n * a.Hkv * D + d);
      to[0] = o[0], to[1] = o[1];
    }
  }
}

extern "C" int pp_kv_read(const void* k_pages, const void* v_pages, const void* k_scales, const void* v_scales, int64_t n_rows,
                          int n_seqs, const int32_t* cu_q, const int32_t* kv_lens, const int32_t* block_table, int max_pages,
                          int num_pages, int page_size, int Hkv, int D, void* k_out, void* v_out, int zero_tail, void* stream) {
  const char* const what = "pp_kv_read";
  int rc = pp_paged_check(what, n_rows, n_seqs, cu_q, kv_lens, block_table, max_pages, k_pages, v_pages, num_pages, page_size, 0,
                          Hkv, D);
  if (rc) return rc;
  PP_REQUIRE(!k_scales == !v_scales, PP_ERR_INVALID, "%s: scales of keys and of values belong together", what);
  if (n_rows == 0) return PP_OK;
  PP_REQUIRE(k_out && v_out, PP_ERR_INVALID, "%s: null pointer", what);
  PP_REQUIRE((((uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, PP_ERR_INVALID, "%s: results not 16-byte aligned", what);
  ReadArgs a = {};
  a.seqs = {cu_q, kv_lens, block_table, (int)n_rows, n_seqs, max_pages, num_pages, paged_log2(page_size)};
  a.k = k_pages, a.v = v_pages, a.k_scales = (const uint8_t*)k_scales, a.v_scales = (const uint8_t*)v_scales;
  a.k_out = (bf16_t*)k_out, a.v_out = (bf16_t*)v_out, a.Hkv = Hkv, a.zero_tail = zero_tail;
  const int vheads = 512 / D;
  a.nkb = (Hkv + 3) / 4, a.nvb = (Hkv + vheads - 1) / vheads;
  const int64_t items = ((n_rows >> 4) + 2 * ((int64_t)n_seqs + 1)) * (a.nkb + a.nvb);
  PP_REQUIRE(items <= 0xffffff, PP_ERR_UNSUPPORTED, "%s: %lld work items (at most 2^24 - 1)", what, (long long)items);
  hipStream_t st = (hipStream_t)stream;
  const unsigned grid = (unsigned)items;
  if (D == 64) {
    if (k_scales) kv_read_kernel<64, true><<<grid, APP_THREADS, 0, st>>>(a);
    else kv_read_kernel<64, false><<<grid, APP_THREADS, 0, st>>>(a);
  } else {
    if (k_scales) kv_read_kernel<128, true><<<grid, APP_THREADS, 0, st>>>(a);
    else kv_read_kernel<128, false><<<grid, APP_THREADS, 0, st>>>(a);
  }
  return pp_check_launch(what);
}
