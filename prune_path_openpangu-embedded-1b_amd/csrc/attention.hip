// Attention of the new tokens of a ragged batch over a paged cache.
//
//   o[i, h] = sum_t p_t v_t,  p = softmax_t(scale q[i, h] . k_t),  t = 0 .. position of token i
//
// in one pass over the cache: running maximum m, running sum l and the accumulated o of a row are
// rescaled by exp(m_old - m_new) when m grows; all three in float32. The query heads of one key head
// are rows of the same tile (row r of a sequence and key head = token r / group, head r % group of
// the group), so the cache is read once for the whole group.
//
// Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T: a row's scores, maximum, sum
// and outputs then stay in one column of the MFMA results, i.e. in the lanes l % 16 (or l % 32) = row,
// and the scores are the second product's right operand without leaving their lane, if the rows of
// the K operand are taken in an order that gives every lane 8 consecutive tokens. The V pages keep a
// channel's tokens next to each other ([page][head][channel][token]), so V^T operands are 16-byte
// loads, like K's.
//
// A cache of 8 bits (fp8.h) is widened to bfloat16, its scales with it, on the way to the matrix cores: the products are those
// over the bfloat16 numbers that it stands for, at half of their bytes from memory. (Products of 8-bit operands would run at
// twice the rate, but take a query or a weight in parts of four bits: two hold a query exactly, while weights below
// 2^-17 of a row's largest would be lost to two.)
//
// With a window, a tile walks the first tokens that stay visible, then the tokens from the group of 16 on in which its first
// row's window begins (AttnTile::at); what lies between is not loaded. Rows mask what is not theirs of the tile's walk.
//
// A workgroup takes one tile of rows of one key head over one range of tokens. Where the tiles alone
// do not fill the GPU, a tile's tokens are cut into ranges ("splits"); the ranges' (m, l, o) go to
// the workspace and attn_join_kernel combines them in order. The cut depends on the tile's own tokens
// and on the arguments alone, so a call gives the same bits every time.
//
// Masked places: their scores are replaced, not added to, and a step that has any multiplies the
// finite part of V only; what is not finite in V goes to the rows that attend it by a second product
// (attn_poison). So stale or foreign data in a page, and a later token's NaN, do not reach a row. A
// row that attends nothing gives zeros, and so does one whose scores are all -inf. An infinity of V
// gives the rows that attend it that infinity; NaN beside its opposite, or where the weight of its
// token underflows in a step without a masked place or in the join of the ranges.
#include <algorithm>
#include <cmath>

#include "fp8.h"
#include "paged.h"

// 16 bytes in registers (a plain vector type: arrays of the struct type were kept in LDS)
typedef uint32_t a_u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ a_u4 a_mk(uint32_t x, uint32_t y, uint32_t z, uint32_t w) { return a_u4{x, y, z, w}; }

typedef short attn_bf16x2 __attribute__((ext_vector_type(2)));
#define ATTN_THREADS 256
#define ATTN_LOW -0x1.fffffep127f  // running maximum before the first score: no finite one is less
// Running maxima from which on the exponent s c - m is taken of the rounded product. One fma leaves what the
// rounding took off m's own product, up to 2^-24 of m: from 2^31 on the row's largest score itself would come
// out infinite or as nothing. (The test costs tiles of 128 rows 0.8 %: 8192 tokens 234.0 us without, 235.7.)
#define ATTN_FAR 0x1p24f

struct AttnArgs {
  PagedSeqs seqs;
  const bf16_t* q;
  int64_t qs[2];  // strides of token and head, in elements
  const bf16_t *k, *v;
  int Hq, Hkv, group;
  float c;        // |scale| * log2(e), not 0 (masked scores are -inf): scores in powers of two
  uint32_t flip;  // the sign of scale, on both halves of a pair of q
  bf16_t* out;
  int zero_tail;
  int splits;         // most ranges of a tile
  int base, behind;   // ranges of a tile, see attn_cut
  float *po, *pml;    // workspace: [row][split][D], [row][split][2]
  int* pns;           // workspace: splits of a row
  int tiles;          // tiles of rows, of every sequence together
  const uint8_t *ks, *vs;  // scales of an 8-bit cache: [page][head][16 tokens]
  int window, sinks;  // tokens that a row attends, itself among them, and first tokens that every row does (window 0: all)
};

// What a workgroup works on.
struct AttnTile {
  int s;         // sequence
  int c0;        // its first row on the token axis
  int r0, nr;    // rows of the tile
  int64_t p0;    // position of the sequence's first new token
  int nt;        // tokens that the tile's last row attends
  int lo, hi;    // tokens of this range
  int ns;        // ranges of the tile (0: nothing is attended)
  // With a window, nt, lo and hi leave out the gap between the first tokens that stay visible and the first that a window
  // reaches: token t of them is token t of the sequence below `keep`, t + gap from there on.
  int keep, gap;
  template <bool WIN>
  __device__ __forceinline__ int at(int t) const { return !WIN || t < keep ? t : t + gap; }
};

// Most ranges of a tile in this call: `behind` in a chunk of one sequence far behind the cache's start. (Asked
// for ahead of everything else where the two differ; the length is read on the device, so the host cannot tell.)
__device__ __forceinline__ int attn_ranges(const AttnArgs& a) {
  if (a.base == a.behind || a.seqs.n_seqs != 1) return a.base;
  return (int64_t)a.seqs.kv_lens[0] >= 2 * (int64_t)a.seqs.n_rows ? a.behind : a.base;
}

// Ranges of a tile that attends nt tokens. It goes by the tokens that are there, not by the table's width,
// which may be any number of times theirs.
template <int R>
__device__ __forceinline__ int attn_cut(const AttnArgs& a, int nt, int ranges) {
  int cut;
  if (R == 16)  // `ranges` of 128 tokens and more, and at least one per 1024; up to 384 tokens the join costs more
    cut = nt <= 384 ? 1 : max(min(ranges, (nt + 127) / 128), nt >> 10);
  else  // of 512 tokens and more
    cut = min(ranges, (nt + 511) / 512);
  return max(1, min(cut, a.splits));
}

// Tile t, of the sequence f. STEP: tokens of a step, which lie on one side of the gap.
template <int R, bool WIN, int STEP>
__device__ __forceinline__ AttnTile attn_tile(const AttnArgs& a, const PagedSeq& f, int64_t t, int split, int ranges) {
  AttnTile w;
  const int g = a.group;
  auto first = [g](int c, int s) { return (int64_t)c * g / R + s; };
  w.s = f.s, w.c0 = f.c0;
  const int len = f.rows;
  const int64_t r0 = (t - first(w.c0, w.s)) * R;
  w.nr = r0 < 0 ? 0 : (int)max((int64_t)0, min((int64_t)R, (int64_t)len * g - r0));  // < 0: offsets out of order
  w.r0 = (int)max((int64_t)0, min(r0, (int64_t)len * g));
  const bool tail = w.s == a.seqs.n_seqs;
  w.p0 = tail ? -(int64_t)len : (int64_t)f.len - len;
  w.nt = (int)max((int64_t)0, min(w.p0 + (w.r0 + max(w.nr, 1) - 1) / g + 1, (int64_t)a.seqs.capacity()));
  w.keep = w.gap = 0;
  if constexpr (WIN) {
    // the first token that the first row's window reaches
    const int start = (int)max((int64_t)0, min(w.p0 + w.r0 / g - a.window + 1, (int64_t)w.nt));
    w.keep = (min(a.sinks, start) + STEP - 1) / STEP * STEP;
    w.gap = max(0, (start & ~15) - w.keep);
    w.nt -= w.gap;
  }
  // equal ranges of whole steps, none of them empty
  const int cut = attn_cut<R>(a, w.nt, ranges);
  const int per = ((w.nt + cut - 1) / cut + 127) / 128 * 128;
  w.ns = w.nt > 0 ? (w.nt + per - 1) / per : 0;
  w.lo = (int)min((int64_t)split * per, (int64_t)w.nt);
  w.hi = min(w.nt, w.lo + per);
  // the same in every lane: said so, or what is computed from them takes vector registers
  for (int* v : {&w.r0, &w.nr, &w.nt, &w.lo, &w.hi, &w.ns}) *v = __builtin_amdgcn_readfirstlane(*v);
  if constexpr (WIN)
    for (int* v : {&w.keep, &w.gap}) *v = __builtin_amdgcn_readfirstlane(*v);
  return w;
}

__device__ __forceinline__ int64_t attn_row(const AttnArgs& a, const AttnTile& w, int h, int r) {
  const int i = (w.r0 + r) / a.group;
  return (int64_t)(w.c0 + i) * a.Hq + h * a.group + (w.r0 + r - i * a.group);
}

// The queries of row r.
__device__ __forceinline__ const bf16_t* attn_query(const AttnArgs& a, const AttnTile& w, int h, int r) {
  const int i = (w.r0 + r) / a.group;
  return a.q + (int64_t)(w.c0 + i) * a.qs[0] + (int64_t)(h * a.group + w.r0 + r - i * a.group) * a.qs[1];
}

// Last position that row r attends.
__device__ __forceinline__ int attn_limit(const AttnArgs& a, const AttnTile& w, int r) {
  return (int)min(w.p0 + (w.r0 + r) / a.group, (int64_t)a.seqs.capacity() - 1);
}

// First position of row r's window (of its place, wherever the table ends).
__device__ __forceinline__ int attn_from(const AttnArgs& a, const AttnTile& w, int r) {
  return (int)max(w.p0 + (w.r0 + r) / a.group - a.window + 1, (int64_t)0);
}

// Rows that attend nothing: zeros (rows of no sequence: only if the call owns the output).
__device__ __forceinline__ void attn_zero(const AttnArgs& a, const AttnTile& w, int h, int D) {
  const bool tail = w.s == a.seqs.n_seqs;
  for (int k = threadIdx.x; k < w.nr * (D / 8); k += ATTN_THREADS) {
    const int r = k / (D / 8), d = 8 * (k - r * (D / 8));
    const int64_t row = attn_row(a, w, h, r);
    if (!tail || a.zero_tail) *(a_u4*)(a.out + row * D + d) = a_mk(0, 0, 0, 0);
    if (a.splits > 1 && d == 0) a.pns[row] = 0;
  }
}

// ------------------------------------------------------------------ masked steps
// Bits 15 and 31 of a word: whether its two elements are not finite (an exponent of ones carries).
__device__ __forceinline__ uint32_t attn_bad2(uint32_t x) { return (x & 0x7f807f80u) + 0x00800080u; }
__device__ __forceinline__ uint32_t attn_bad(const a_u4 v) {
  return attn_bad2(v[0]) | attn_bad2(v[1]) | attn_bad2(v[2]) | attn_bad2(v[3]);
}
__device__ __forceinline__ uint32_t attn_clean1(uint32_t x) { return (x & 0x7f80u) == 0x7f80u ? 0u : x; }
__device__ __forceinline__ a_u4 attn_clean(a_u4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = attn_clean1(v[i] & 0xffffu) | (attn_clean1(v[i] >> 16) << 16);
  return v;
}
// +inf, -inf and NaN as 1, 2^8 and 2^16 (everything else 0): a sum of up to 64 of them tells how many
// of each there are, exactly, in float32.
__device__ __forceinline__ uint32_t attn_code1(uint32_t x) {
  if ((x & 0x7f80u) != 0x7f80u) return 0u;
  return (x & 0x7fu) ? 0x4780u : (x & 0x8000u) ? 0x4380u : 0x3f80u;
}
__device__ __forceinline__ a_u4 attn_code(a_u4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = attn_code1(v[i] & 0xffffu) | (attn_code1(v[i] >> 16) << 16);
  return v;
}
__device__ __forceinline__ float attn_poison(float o, float code) {
  const uint32_t n = (uint32_t)code;
  if (n == 0) return o;
  const bool up = n & 0xffu, down = (n >> 8) & 0xffu;
  if ((n >> 16) || (up && down)) return __uint_as_float(0x7fc00000u);
  return o + __uint_as_float(up ? 0x7f800000u : 0xff800000u);
}

// 1 for every attended of 8 tokens (bits of `seen`), as an operand.
__device__ __forceinline__ a_u4 attn_ones(uint32_t seen) {
  a_u4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    v[j] = ((seen >> (2 * j)) & 1 ? 0x3f80u : 0u) | ((seen >> (2 * j + 1)) & 1 ? 0x3f800000u : 0u);
  return v;
}


// 16 values of 8 bits times their scale, as two operands.
__device__ __forceinline__ void attn_wide(const a_u4 v, float scale, a_u4& lo, a_u4& hi) {
  lo = a_mk(fp8_bf16<false>(v[0], scale), fp8_bf16<true>(v[0], scale), fp8_bf16<false>(v[1], scale), fp8_bf16<true>(v[1], scale));
  hi = a_mk(fp8_bf16<false>(v[2], scale), fp8_bf16<true>(v[2], scale), fp8_bf16<false>(v[3], scale), fp8_bf16<true>(v[3], scale));
}

// The bf16 value below p (0 for 0), as a float's bits.
__device__ __forceinline__ uint32_t attn_upper(float p) {
  return __builtin_elementwise_sub_sat(__float_as_uint(p), 1u) & 0xffff0000u;
}

// max(a, b, c), NaN if one is: one v_maximum3_f32 (fmaxf, which passes NaN over, first makes each operand
// a quiet value).
__device__ __forceinline__ float attn_max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}
// l plus both halves of a pair of bf16 values: one v_dot2_f32_bf16
__device__ __forceinline__ float attn_sum2(uint32_t pair, float l) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(attn_bf16x2, pair), __builtin_bit_cast(attn_bf16x2, 0x3f803f80u), l, false);
}
__device__ __forceinline__ float attn_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// v_mfma_f32_16x16x32_bf16: A lane l holds row l % 16, k = 8 (l / 16) .. + 7; B lane l column l % 16,
// the same k; D lane l, element i is row 4 (l / 16) + i, column l % 16.
__device__ __forceinline__ f32x4_t mfma16(const a_u4 a, const a_u4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ f32x16_t mfma32a(const a_u4 a, const a_u4 b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// ------------------------------------------------------------------ few rows
// Up to 16 rows of one key head; the cache bounds it. The four waves take alternate steps of 32
// tokens, each with its own m, l and o, and join them at the end through LDS. K and V operands come
// straight from memory into registers. The next step's K is asked for once the present one's scores
// are computed, its V after the second product, so a wave always has one of the two in flight with
// one set of registers.
// K operand row m of block b (16 tokens) is token 8 (m / 4) + 4 b + m % 4 of the step, which leaves
// lane group g = lane / 16 with the scores of tokens 8 g .. 8 g + 7: its k of the second product.
// P enters as a sum of two bf16 values, its upper bits and what is left, rounded (2^-15 of P at most): the
// second product costs nothing next to the loads. The upper part is below P, so that an infinity of V in an
// attended place gives that infinity: nothing left, or what is left of an upper part rounded up, would make it
// NaN.
// Measured, 12 heads of 128: one token on each of 64 sequences of 8192 557 us (3.2 GB, 5.8 TB/s, where a
// large copy reaches 4.9), of 1 to 8192 tokens 270 us (5.6 TB/s); one sequence of 1152 tokens 8.9 us with
// the join's 3.5, chains of offsets, table, K and join rather than bytes.
// 8 bits: a lane's 16 bytes are 16 channels of a K row, two operands of it (the queries go the same way), and 16 tokens, a
// block, of a V channel: steps of 64 tokens with the same registers in flight, one scale a lane for each of K and V.
// 64 sequences of 8192 tokens 283 us (1.6 GB, 5.7 TB/s), of 1 to 8192 150, one of 1152 9.0 with the join. (219 registers, two
// waves a SIMD: the widened operands of one piece at a time; all at once spilled.)
// A window of 1000 and 4 first tokens, 32 sequences anywhere in 16384, 24 heads on 8: 18.4 us (64 MB of 8 bits: five steps a
// wave behind the chain of loads).
// A lane's sequence of up to 64: its first row, its rows; and the first row of no sequence.
struct AttnLane {
  int c, rows, len, end;
};
__device__ __forceinline__ AttnLane attn_lane(const AttnArgs& a) {
  const int n = a.seqs.n_seqs, lane = threadIdx.x & 63, s = min(lane, n - 1);
  const int this_q = a.seqs.cu_q[s], next_q = a.seqs.cu_q[s + 1], len = a.seqs.kv_lens[s], last_q = a.seqs.cu_q[n];
  paged_asked();
  auto row = [&](int c) { return min(max(c, 0), a.seqs.n_rows); };
  AttnLane x;
  x.c = s == 0 ? 0 : row(this_q), x.end = row(last_q), x.len = len;
  x.rows = lane < n ? max(row(next_q) - x.c, 0) : 0;
  return x;
}
// The sequence of lane l, the rows of none if l < 0.
__device__ __forceinline__ PagedSeq attn_of(const AttnArgs& a, const AttnLane& x, int l) {
  PagedSeq f;
  const int at = max(l, 0), end = __builtin_amdgcn_readfirstlane(x.end);
  f.s = l < 0 ? a.seqs.n_seqs : l;
  f.c0 = l < 0 ? end : __builtin_amdgcn_readlane(x.c, at);
  f.rows = l < 0 ? a.seqs.n_rows - end : __builtin_amdgcn_readlane(x.rows, at);
  f.len = l < 0 ? 0 : __builtin_amdgcn_readlane(x.len, at);
  return f;
}
// The sum of v over the lanes up to this one.
__device__ __forceinline__ int attn_scan(int v) {
#define ATTN_SCAN(ctrl, rows) v += __builtin_amdgcn_update_dpp(0, v, ctrl, rows, 0xf, false)
  ATTN_SCAN(0x111, 0xf);
  ATTN_SCAN(0x112, 0xf);
  ATTN_SCAN(0x114, 0xf);
  ATTN_SCAN(0x118, 0xf);
  ATTN_SCAN(0x142, 0xa);
  ATTN_SCAN(0x143, 0xc);
#undef ATTN_SCAN
  return v;
}

// Tile u of those that have rows, -1: none, and its sequence. The numbers of tiles have gaps (a sequence takes one more than it
// may need); of up to 64 sequences those with rows come first, so that their workgroups are the first ones of the grid and
// find a CU each where there are that many: workgroups of the gaps among them held places for the moment in which the last
// ones were given out, two to a CU while others went idle (32 single tokens, 24 heads on 8, a window of 1000: 18.7 us instead of
// 22.8 over 8 bits, 24.4 instead of 31.7 over 16; 64 of 500 tokens, 12 heads, 22.8 instead of 24.3).
__device__ __forceinline__ int attn_filled(const AttnArgs& a, int u, PagedSeq& f) {
  const int n = a.seqs.n_seqs;
  if (n < 1 || n > 64) {
    f = paged_find(a.seqs, u, [&](int c, int s) { return (int64_t)c * a.group / 16 + s; });
    return u;
  }
  const AttnLane x = attn_lane(a);
  auto first = [&](int c, int s) { return (int)((int64_t)c * a.group / 16 + s); };
  const int tiles = (int)(((int64_t)x.rows * a.group + 15) / 16), upto = attn_scan(tiles);
  const int all = __builtin_amdgcn_readlane(upto, 63);
  const uint64_t mine = __ballot(u < upto && u >= upto - tiles);
  const int l = mine != 0 ? __builtin_ctzll(mine) : -1;
  f = attn_of(a, x, l);
  if (l < 0) return first(f.c0, n) + u - all;  // (beyond its rows: a tile without any)
  return first(f.c0, l) + u - __builtin_amdgcn_readlane(upto - tiles, l);
}

template <int D, bool EIGHT, bool WIN>
__global__ __launch_bounds__(ATTN_THREADS, EIGHT ? 2 : 3) void attn_few_kernel(AttnArgs a) {
  constexpr int R = 16, KS = D / 32, MB = D / 16, OS = D + 4;
  constexpr int TOK = EIGHT ? 16 : 8, ST = 4 * TOK, KB = TOK / 4;  // tokens of a lane, of a step, blocks of a step's K
  constexpr int KL = EIGHT ? D / 64 : KS;                          // 16-byte pieces of a K row to a lane
  __shared__ float o_s[4][R][OS];
  __shared__ float ml_s[4][R][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, g = lane >> 4;
  // Items are (split, tile, head), the heads fastest: a tile's later ranges, which many do not have, behind every
  // tile's first. (Next to them, ranges of one number met on few of the XCDs: 64 sequences of 2000 tokens in a
  // table of eight ranges 607 us instead of 142.) The last tile, as a rule of no sequence, behind everything: the
  // workgroups that have work are the first ones, one to a CU if they are few (one token at 8191 15 us, 19
  // without). Workgroup b runs on XCD b % 8: ranges of one number begin half way round from those before, for
  // where every other tile is empty and half of the XCDs would have all the work (32 sequences of two rows, 4
  // heads, 119 us instead of 140).
  const int items = (a.tiles - 1) * a.Hkv, most = items * a.splits, b = blockIdx.x;
  const int split = b < most ? b / items : (b - most) / a.Hkv, turn = split * (items - 4) & 7;
  const int item = b < most ? (b - split * items + turn) % items : items + (b - most) % a.Hkv, h = item % a.Hkv;
  PagedSeq seq;
  const int tile = __builtin_amdgcn_readfirstlane(attn_filled(a, item / a.Hkv, seq));
  for (int* v : {&seq.s, &seq.c0, &seq.rows, &seq.len}) *v = __builtin_amdgcn_readfirstlane(*v);
  const AttnTile w = attn_tile<R, WIN, ST>(a, seq, tile, split, a.base);
  if (w.nr <= 0) return;
  if (w.ns == 0) {
    if (split == 0) attn_zero(a, w, h, D);
    return;
  }
  if (split >= w.ns) return;

  const int ps = 1 << a.seqs.lp;
  const int gk = TOK * (col >> 2), gv = TOK * g;  // the lane's tokens of K and of V, within a step
  int ek, ev;                                 // their table entries
  int pk, pv;                                 // their pages, -1: none
  int pc;                                     // the present V's
  a_u4 kf[KB][KL], vf[MB];
  uint32_t sk = 0, sv = 0;                    // 8 bits: the scales of what kf and vf hold
  // Loads are asked for without a branch, of the last row or entry where there is none: with one, the
  // wait for each stands where the two sides meet.
  const int32_t* const table = a.seqs.table + (int64_t)w.s * a.seqs.max_pages;
  const int last_entry = w.at<WIN>(w.hi - 1) >> a.seqs.lp;
  auto entries = [&](int t) {
    const int at = w.at<WIN>(t);
    ek = table[min((at + gk) >> a.seqs.lp, last_entry)];
    ev = table[min((at + gv) >> a.seqs.lp, last_entry)];
  };
  auto pages = [&](int t) {
    pk = t + gk < w.hi ? a.seqs.page(ek) : -1;
    pv = t + gv < w.hi ? a.seqs.page(ev) : -1;
  };
  // places without a page read page 0, and are masked
  auto load_k = [&](int t) {
    const int64_t row = (((int64_t)max(pk, 0) * a.Hkv + h) << a.seqs.lp) + ((w.at<WIN>(t) + gk) & (ps - 1));
    if constexpr (EIGHT) {
      const uint8_t* kp = (const uint8_t*)a.k + (row + (col & 3)) * D + 16 * g;
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int s = 0; s < KL; ++s) kf[b][s] = *(const a_u4*)(kp + 4 * b * D + 64 * s);
      sk = a.ks[row >> 4];
    } else {
      const bf16_t* kp = a.k + (row + (col & 3)) * D + 8 * g;
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int s = 0; s < KL; ++s) kf[b][s] = *(const a_u4*)(kp + 4 * b * D + 32 * s);
    }
  };
  auto at_v = [&](int page, int t) {
    return a.v + ((((int64_t)max(page, 0) * a.Hkv + h) * D + col) << a.seqs.lp) + ((w.at<WIN>(t) + gv) & (ps - 1));
  };
  auto load_v = [&](int t) {
    pc = pv;
    if constexpr (EIGHT) {
      const int64_t block = ((((int64_t)max(pv, 0) * a.Hkv + h) << a.seqs.lp) + ((w.at<WIN>(t) + gv) & (ps - 1))) >> 4;
      const a_u4* vp = (const a_u4*)((const uint8_t*)a.v + block * (16 * D)) + col;
#pragma unroll
      for (int b = 0; b < MB; ++b) vf[b] = vp[16 * b];
      sv = a.vs[block];
    } else {
      const bf16_t* vp = at_v(pv, t);
#pragma unroll
      for (int b = 0; b < MB; ++b) vf[b] = *(const a_u4*)(vp + ((int64_t)(16 * b) << a.seqs.lp));
    }
  };
  int t = w.lo + ST * wave;
  entries(t);
  a_u4 qf[KS];
  const bool in = col < w.nr;
  const int limit = in ? attn_limit(a, w, col) : a.seqs.capacity();
  // (8 bits: a lane's 16 channels of K are two operands, so the queries' go the same way)
  const bf16_t* const src = attn_query(a, w, h, min(col, w.nr - 1)) + TOK * g;
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = *(const a_u4*)(src + (EIGHT ? 64 * (s >> 1) + 8 * (s & 1) : 32 * s));
  paged_asked();
  pages(t);
  entries(t + 4 * ST);
  load_k(t);
  load_v(t);
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = in ? qf[s] ^ a.flip : a_mk(0, 0, 0, 0);
  const int low = attn_limit(a, w, 0);  // every row attends the tokens up to here
  // windows: the row's first token, and the first that every row's holds
  const int from = WIN ? attn_from(a, w, min(col, w.nr - 1)) : 0, high = WIN ? attn_from(a, w, w.nr - 1) : 0;

  f32x4_t o[MB];
  float m = ATTN_LOW, l = 0.0f;
#pragma unroll
  for (int b = 0; b < MB; ++b) o[b] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  for (; t < w.hi; t += 4 * ST) {
    const int rt = w.at<WIN>(t);  // the step's first position
    pages(t + 4 * ST);
    entries(t + 8 * ST);
    f32x4_t s[KB];
    const float fk = fp8_factor(sk), fv = fp8_factor(sv);
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      s[b] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int q = 0; q < KL; ++q) {
        if constexpr (EIGHT) {
          a_u4 k0, k1;
          attn_wide(kf[b][q], fk, k0, k1);
          s[b] = mfma16(k0, qf[2 * q], s[b]);
          s[b] = mfma16(k1, qf[2 * q + 1], s[b]);
        } else {
          s[b] = mfma16(kf[b][q], qf[q], s[b]);
        }
      }
    }
    const bool more = t + 4 * ST < w.hi;
    if (more) load_k(t + 4 * ST);
    // whether a place of the step is masked for any row (wave-uniform)
    const bool part = rt + ST - 1 > low || t + ST > w.hi || (WIN && rt < high) || __ballot(pc < 0) != 0;
    bool bad = false;
    if (part) {
      uint32_t any = 0;
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        if constexpr (EIGHT) any |= fp8_bad(vf[b][0]) | fp8_bad(vf[b][1]) | fp8_bad(vf[b][2]) | fp8_bad(vf[b][3]);
        else any |= attn_bad(vf[b]);
      }
      bad = __ballot((any & (EIGHT ? 0x80808080u : 0x80008000u)) != 0 || (EIGHT && sv > FP8_HIGH)) != 0;
      if (!EIGHT && bad) {
#pragma unroll
        for (int b = 0; b < MB; ++b) vf[b] = attn_clean(vf[b]);
      }
    }
    float p[TOK];
#pragma unroll
    for (int j = 0; j < TOK; ++j) p[j] = s[j >> 2][j & 3];
    uint32_t seen = (1u << TOK) - 1;
    if (part) {
      asm volatile("");  // a branch: few steps have one
      seen = 0;
#pragma unroll
      for (int j = 0; j < TOK; ++j) {
        const int at = rt + gv + j;
        const bool in = pc >= 0 && at <= limit && t + gv + j < w.hi && (!WIN || at >= from || at < a.sinks);
        seen |= in ? 1u << j : 0u;
        p[j] = in ? p[j] : -__builtin_inff();
      }
    }
    float top = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
    if constexpr (EIGHT)
      top = fmaxf(top, fmaxf(fmaxf(fmaxf(p[8], p[9]), fmaxf(p[10], p[11])), fmaxf(fmaxf(p[12], p[13]), fmaxf(p[14], p[15]))));
    top = fmaxf(top, pl_xor16f(top, lane));
    top = fmaxf(top, pl_xor32f(top, lane));
    const float mn = fmaxf(m, top * a.c), shrink = attn_exp2(m - mn);
    m = mn;
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < TOK; ++j) {
      p[j] = attn_exp2(__fmul_rn(p[j], a.c) - mn);  // (in two steps, see ATTN_FAR: the loads hide the second)
      sum += p[j];
    }
    l = __fmaf_rn(l, shrink, sum);
    uint32_t hi[TOK / 2], lo[TOK / 2];
#pragma unroll
    for (int j = 0; j < TOK / 2; ++j) {
      const uint32_t u = attn_upper(p[2 * j]), v = attn_upper(p[2 * j + 1]);
      hi[j] = (u >> 16) | v;
      lo[j] = f32_to_bf16x2(p[2 * j] - __uint_as_float(u), p[2 * j + 1] - __uint_as_float(v));
    }
    const a_u4 ph = a_mk(hi[0], hi[1], hi[2], hi[3]), pl = a_mk(lo[0], lo[1], lo[2], lo[3]);
    if constexpr (EIGHT) {
      const a_u4 ph2 = a_mk(hi[4], hi[5], hi[6], hi[7]), pl2 = a_mk(lo[4], lo[5], lo[6], lo[7]);
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        a_u4 v0, v1, all0, all1;
        attn_wide(vf[b], fv, v0, v1);
        if (bad) {  // only the finite part of V, and what is not finite for the rows that attend it
          asm volatile("");
          all0 = v0, all1 = v1;
          v0 = attn_clean(v0), v1 = attn_clean(v1);
        }
        o[b] *= shrink;
        o[b] = mfma16(v0, ph, o[b]);
        o[b] = mfma16(v1, ph2, o[b]);
        o[b] = mfma16(v0, pl, o[b]);
        o[b] = mfma16(v1, pl2, o[b]);
        if (bad) {
          asm volatile("");
          f32x4_t code = mfma16(attn_code(all0), attn_ones(seen), f32x4_t{0.0f, 0.0f, 0.0f, 0.0f});
          code = mfma16(attn_code(all1), attn_ones(seen >> 8), code);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[b][i] = attn_poison(o[b][i], code[i]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        o[b] *= shrink;
        o[b] = mfma16(vf[b], ph, o[b]);
        o[b] = mfma16(vf[b], pl, o[b]);
      }
      if (bad) {  // what was taken out of V, read again, for the rows that attend it
        const a_u4 one = attn_ones(seen);
        const bf16_t* vp = at_v(pc, t);
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          const a_u4 x = *(const a_u4*)(vp + ((int64_t)(16 * b) << a.seqs.lp));
          const f32x4_t code = mfma16(attn_code(x), one, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
          for (int i = 0; i < 4; ++i) o[b][i] = attn_poison(o[b][i], code[i]);
        }
      }
    }
    if (more) load_v(t + 4 * ST);
  }

  // the four waves' rows joined
  l += pl_xor16f(l, lane);
  l += pl_xor32f(l, lane);
  if (g == 0) ml_s[wave][col][0] = m, ml_s[wave][col][1] = l;
#pragma unroll
  for (int b = 0; b < MB; ++b) *(f32x4_t*)&o_s[wave][col][16 * b + 4 * g] = o[b];
  __syncthreads();
  for (int k = tid; k < w.nr * (D / 8); k += ATTN_THREADS) {
    const int r = k / (D / 8), d = 8 * (k - r * (D / 8));
    float mm = ml_s[0][r][0];
#pragma unroll
    for (int i = 1; i < 4; ++i) mm = fmaxf(mm, ml_s[i][r][0]);
    float sum = 0.0f, acc[8] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = attn_exp2(ml_s[i][r][0] - mm);
      sum = __fmaf_rn(ml_s[i][r][1], f, sum);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = __fmaf_rn(o_s[i][r][d + j], f, acc[j]);
    }
    const int64_t row = attn_row(a, w, h, r);
    if (w.ns == 1) {
      const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
      *(a_u4*)(a.out + row * D + d) = a_mk(f32_to_bf16x2(acc[0] * inv, acc[1] * inv), f32_to_bf16x2(acc[2] * inv, acc[3] * inv),
                                                  f32_to_bf16x2(acc[4] * inv, acc[5] * inv), f32_to_bf16x2(acc[6] * inv, acc[7] * inv));
    } else {
      float* to = a.po + (row * a.splits + split) * D + d;
      *(float4*)to = make_float4(acc[0], acc[1], acc[2], acc[3]);
      *(float4*)(to + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
      if (d == 0) *(float2*)(a.pml + (row * a.splits + split) * 2) = make_float2(mm, sum);
    }
    if (a.splits > 1 && split == 0 && d == 0) a.pns[row] = w.ns;
  }
}

// ------------------------------------------------------------------ many rows
// 128 rows of one key head, 32 to each of four waves. Steps of 64 tokens: K [64][D] and V^T [D][64]
// are copied into one of two LDS buffers without passing through registers, the next step's while
// the present one is computed (one barrier a step). Row m of the K tile is the token whose number
// within its 16 has bits 2 and 3 of m swapped, which leaves lane half e = lane / 32 with the scores of
// tokens 16 b + 8 e .. + 7: its k of the second product. The 16-byte chunks of an LDS row are
// permuted, so that the 16 lanes that read at a time, on 16 different rows, meet all 64 banks: in rows
// of 256 bytes chunk c sits at place c ^ (row % 16), in rows of 128 at c ^ (row / 2 % 8).
// P enters the second product as one bf16 value, and l sums the values as they are rounded, so that weights
// still add up to 1: 2^-8 of a weight at most, 3e-4 of a result in the 2-norm (5e-4 with the sum of the values
// before) beside the 1.7e-3 of its own rounding to bf16. Two parts, as above, would take 512 clocks more of the
// matrix cores a step.
// Two workgroups share a CU at D = 128, and a wave's step takes 4300 clocks, where its products take 1024 and
// its vector instructions issue for 1200: 390 at the barrier, 1080 until the 8 copies are issued (30
// bytes a clock and CU, with the other workgroup's), 910 in the first product, 460 for the maximum, 1160 in the
// second product, 340 for the sums. The counters have the matrix cores busy for 47 %, the vector units for
// 50, LDS for 24 without conflicts, and 86 % of the copies' lines in L2. A part that was shortened
// came back as waiting elsewhere: copies between the products (8192 tokens 245 us instead of 233), V's
// behind the first product (242; 512 tokens at 30000 129 instead of 137), sums beside the last products,
// 256 rows on eight waves with the second product of one half beside the first of the other (236) or on
// four, one a SIMD (319), no priorities (232).
// Measured: 12 heads of 128, a prompt of 8192 tokens 238 us (870 TFLOP/s; as much in pages of 64), of 4096 85 us
// (605), of 2048 37 us, 7 of them the join's; 512 new tokens at 30000 131 us (730).
// 8 bits: the next step's 16 bytes of K and V to each thread are asked for before the present step's products, widened and stored
// to LDS behind them: 8192 tokens 237 us, 4096 84, 512 at 30000 127.
// A window of 1024 and 4 first tokens, 8192 tokens: 87 us (550 TFLOP/s): 19 steps of 64 tokens a tile, five of them with
// masked places (three of a wave's), and three tiles a CU for two places.
#define ATTN_ROWS 128

// 16 bytes per lane from memory into LDS at lds + 16 lane, by the copy path that does not pass through
// registers. The compiler does not know of it: attn_landed() is what waits, for every copy that was
// asked for, before the workgroup's barrier.
typedef __attribute__((address_space(3))) void attn_lds_t;
__device__ __forceinline__ uint32_t attn_lds(void* p) { return (uint32_t)(uintptr_t)(attn_lds_t*)p; }
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 named as clobbered: the compiler sets it anew for each use of its own
__device__ __forceinline__ void attn_copy(const void* from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void attn_landed() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

#define ATTN_KT 64
#define ATTN_SLACK 8.0f

// The u-th tile, -1: none, and its sequence: the last ones, which attend most, first. Of 2 to 64 sequences whose longest walks differ
// by more than a quarter (as the caches do, or as a window and the first tokens leave of them) those with the longest first, so
// that no long tile begins when the others end: a lane has one sequence, and finds the tiles in front of its own, each wave for
// 16 of the sequences (lds: 256 numbers). There, and with a window, the tiles that have rows come before the gaps in the numbers,
// which otherwise hold places while the last of them are given out: 30 chunks of 200 tokens at 1050 to 1500, 12 heads of 64,
// 60 us with the gaps in between, 46 without; 49 in the batch's order. (Sorted in every wave for all the sequences, one at a
// time: 63 chunks of 64 at 670 to 1000, 12 heads of 128, 86 us, like this 79, in the batch's order 80.) Without a window
// sequences that are alike keep the order of the numbers: behind the tiles the gaps make 40 chunks of 128 at 1400 113 -> 81 us, but 63
// of 64 at 4000 302 -> 314. With windows of 1024 and 4 first tokens, in this order, in that of the numbers, by the caches' lengths
// with the gaps in between: 40 chunks of 100 at 800 to 8000, 12 heads of 64, 40, 49, 54 us; 63 of 64 at 2000 to 4000, 12 heads of
// 128, 110, 107, 116, over 8 bits 84, 90, 100.
// (us in this order and in the reverse of the batch's, caches of 16 bits, 12 heads of 128: nine sequences, chunks of up to 700 and
// single tokens, 78 / 92; 20 chunks of up to 600 at up to 4000 160 / 176; eight prompts of up to 3000 62 / 72; a chunk of 900 at
// 8000 and 63 single tokens 212 / 306 if the chunk is the batch's first, 211 / 211 if it is its last.)
template <bool WIN>
__device__ __forceinline__ int attn_order(const AttnArgs& a, int u, int* lds, PagedSeq& f) {
  const int n = a.seqs.n_seqs, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  auto first = [&](int c, int s) { return (int)((int64_t)c * a.group / ATTN_ROWS + s); };  // tile of row c of sequence s
  const int t = a.tiles - 1 - u;
  if (t < 0) return -1;
  if (n < 2 || n > 64) {
    f = paged_find(a.seqs, t, first);
    return t;
  }
  const AttnLane x = attn_lane(a);
  const int tiles = (int)(((int64_t)x.rows * a.group + ATTN_ROWS - 1) / ATTN_ROWS);
  // by walks (up to 2^25; 0: no rows), then by numbers: no two keys are the same
  const int walk = WIN ? (int)min((int64_t)a.window + a.sinks + ATTN_ROWS, (int64_t)(1 << 25) - 1) : (1 << 25) - 1;
  const uint32_t key = (tiles ? (uint32_t)min(max(x.len, 1), walk) << 6 : 0u) | (63 - lane);
  const uint32_t most = (uint32_t)wave_max((float)(key >> 6)), least = (uint32_t)-wave_max(tiles ? -(float)(key >> 6) : -0x1p26f);
  const bool uneven = most >= least && most - least > most / 4;  // (the same in all waves: they meet at the barriers)
  if (WIN || uneven) {
    const int upto = attn_scan(tiles), all = __builtin_amdgcn_readlane(upto, 63);
    int before = all - upto;  // tiles in front of the sequence's: of those behind it in the batch
    if (uneven) {
      int part = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t k = __builtin_amdgcn_readlane(key, 16 * wave + i);
        const int m = __builtin_amdgcn_readlane(tiles, 16 * wave + i);
        part += k > key ? m : 0;
      }
      lds[64 * wave + lane] = part;
      __syncthreads();
      before = (lds[lane] + lds[64 + lane]) + (lds[128 + lane] + lds[192 + lane]);
      __syncthreads();
    }
    const uint64_t mine = __ballot(u >= before && u < before + tiles);
    const int l = mine != 0 ? __builtin_ctzll(mine) : -1;
    f = attn_of(a, x, l);
    if (l < 0) return first(f.c0, n) + u - all;  // behind all of them the rows of no sequence (beyond these: a tile without any)
    return first(f.c0, l) + __builtin_amdgcn_readlane(before + tiles - 1, l) - u;
  }
  const int s = min(lane, n - 1), lo = first(x.c, s), tail = first(x.end, n);
  const int next = __shfl(lo, min(lane + 1, n - 1)), count = lane < n ? max((s + 1 < n ? next : tail) - lo, 0) : 0;
  const uint64_t mine = __ballot(t >= lo && t < lo + count);
  f = attn_of(a, x, mine != 0 ? __builtin_ctzll(mine) : -1);
  return t;
}

template <int D, bool EIGHT, bool WIN>
__global__ __launch_bounds__(ATTN_THREADS, D == 64 ? 3 : 2) void attn_many_kernel(AttnArgs a) {
  constexpr int KC = D / 8, NK = ATTN_KT * KC / ATTN_THREADS, NV = D * (ATTN_KT / 8) / ATTN_THREADS, MB = D / 32;
  __shared__ a_u4 k_s[2][ATTN_KT * KC];
  __shared__ a_u4 v_s[2][D * (ATTN_KT / 8)];
  __shared__ int bad_s[2];  // first token of the buffer's step if V there was not finite
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, e = lane >> 5;
  // Items are (tile, split, head): the tiles that attend most first, and the heads fastest.
  // Workgroup b runs on XCD b % 8, so an XCD meets only the key heads of one remainder (of 8, or of
  // what 8 and their number have in common), whose K and V its L2 then holds.
  // The ranges that the call does have are next to each other, those that it does not behind everything: among
  // them, they left half of the XCDs with most of the work (4096 tokens at 8000 458 us instead of 306).
  const int ranges = max(1, min(attn_ranges(a), a.splits));
  const int h = blockIdx.x % a.Hkv, rest = blockIdx.x / a.Hkv, split = rest % ranges, u = rest / ranges;
  PagedSeq seq;
  const int tile = __builtin_amdgcn_readfirstlane(attn_order<WIN>(a, u, (int*)k_s, seq));
  if (tile < 0) return;
  for (int* v : {&seq.s, &seq.c0, &seq.rows, &seq.len}) *v = __builtin_amdgcn_readfirstlane(*v);
  const AttnTile w = attn_tile<ATTN_ROWS, WIN, ATTN_KT>(a, seq, tile, split, ranges);
  if (w.nr <= 0) return;
  if (w.ns == 0) {
    if (split == 0) attn_zero(a, w, h, D);
    return;
  }
  if (split >= w.ns) return;

  const int r = 32 * wave + col;
  const bool in = r < w.nr, busy = 32 * wave < w.nr;
  const int limit = in ? attn_limit(a, w, r) : 0x7fffffff;
  // tokens that every row of the wave attends, and that any does
  const int low = busy ? attn_limit(a, w, 32 * wave) : 0, top = busy ? attn_limit(a, w, min(32 * wave + 31, w.nr - 1)) : -1;
  // windows: the row's first token, the first that any of the wave's rows attends, that all of the wave's do, all of the tile's
  const int from = WIN ? attn_from(a, w, min(r, w.nr - 1)) : 0, bottom = WIN && busy ? attn_from(a, w, 32 * wave) : 0;
  const int high = WIN && busy ? attn_from(a, w, min(32 * wave + 31, w.nr - 1)) : 0, high0 = WIN ? attn_from(a, w, w.nr - 1) : 0;
  const int ps = 1 << a.seqs.lp;
  // the thread's 16-byte chunk of each K copy (row krow of its 16 or 32) and of each V copy (channel
  // vrow of 32): its place in LDS is tid, so the swizzle is in what it reads
  const int krow = tid / KC, vrow = tid / 8, vc = (tid % 8) ^ ((vrow >> 1) & 7);
  const int kc = (tid % KC) ^ (KC == 16 ? krow & 15 : (krow >> 1) & 7);
  const int k16 = KC == 16 ? 0 : wave >> 1;  // group of 16 rows, at D = 64
  const uint32_t koff = (((krow & 3) | ((krow & 4) << 1) | ((krow & 8) >> 1)) * D + 8 * kc) * 2;  // its row's token
  // The page of the lane's group of 16 tokens, vc / 2, of a step, -1: none: of the present step and the
  // next. Lanes 0 .. 7 have vc = lane ^ of_odd: lane 2 j ^ of_odd has group j's.
  const int of_odd = EIGHT ? 0 : 4 * (wave & 1), group = EIGHT ? (lane >> 1) & 3 : vc >> 1;
  int pg, pn, en;  // en: the table entry of the step after the next
  const int32_t* const table = a.seqs.table + (int64_t)w.s * a.seqs.max_pages;
  const int last_entry = w.at<WIN>(w.hi - 1) >> a.seqs.lp;
  // The entry is asked for without a branch, beyond the range for its last one's: with one, the wait for it
  // stood where the two sides meet, behind the copies, and so for all of them (8192 tokens 248 us).
  auto entry = [&](int t) { en = table[min((w.at<WIN>(t) + 16 * group) >> a.seqs.lp, last_entry)]; };
  auto page = [&](int t) { return t + 16 * group < w.hi ? a.seqs.page(en) : -1; };
  const uint32_t k_lds = attn_lds(&k_s[0][64 * wave]), v_lds = attn_lds(&v_s[0][64 * wave]);
  // 8 bits: what a thread copies goes through its registers, asked for a step ahead and widened to the same places: 16
  // channels of K row 32 i + tid / 8 (at D = 64 row tid / 4), and 16 tokens, of group 2 i + tid / 128 (tid / 64), of V channel
  // tid % D.
  constexpr int N8 = D / 64, C8 = D / 16;
  a_u4 k8[N8], v8[N8];
  uint32_t sk8[N8], sv8[N8];
  const int m8 = tid / C8;  // its first K row
  auto group_k = [&](int i) { return D == 128 ? 2 * i + (wave >> 1) : wave; };
  auto ask = [&](int t) {
    const int at = w.at<WIN>(t);
#pragma unroll
    for (int i = 0; i < N8; ++i) {
      const int j = group_k(i), p = __builtin_amdgcn_readlane(pn, 2 * j);
      const int64_t first = (((int64_t)max(p, 0) * a.Hkv + h) << a.seqs.lp) + ((at + 16 * j) & (ps - 1));
      const int row = (m8 & 3) | ((m8 & 4) << 1) | ((m8 & 8) >> 1);
      k8[i] = *(const a_u4*)((const uint8_t*)a.k + (first + row) * D + 16 * (tid % C8));
      v8[i] = ((const a_u4*)((const uint8_t*)a.v + first * D))[tid % D];
      sk8[i] = a.ks[first >> 4], sv8[i] = a.vs[first >> 4];
    }
  };
  auto widen = [&](int buf) {
#pragma unroll
    for (int i = 0; i < N8; ++i) {
      const int m = m8 + 32 * i, sw = KC == 16 ? m & 15 : (m >> 1) & 7, c = 2 * (tid % C8), ch = tid % D, vs = (ch >> 1) & 7, j = group_k(i);
      a_u4 x, y;
      attn_wide(k8[i], fp8_factor(sk8[i]), x, y);
      k_s[buf][m * KC + (c ^ sw)] = x, k_s[buf][m * KC + ((c + 1) ^ sw)] = y;
      attn_wide(v8[i], fp8_factor(sv8[i]), x, y);
      v_s[buf][ch * 8 + ((2 * j) ^ vs)] = x, v_s[buf][ch * 8 + ((2 * j + 1) ^ vs)] = y;
    }
  };
  auto load = [&](int t, int buf) {  // places without a page read page 0, and are masked
    if constexpr (EIGHT) {
      ask(t);
      return;
    }
    t = w.at<WIN>(t);
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int j = KC == 16 ? i : 2 * i + k16;  // its group of 16 tokens
      const int p = __builtin_amdgcn_readlane(pn, (2 * j) ^ of_odd);
      const bf16_t* base = a.k + ((((int64_t)max(p, 0) * a.Hkv + h) << a.seqs.lp) + ((t + 16 * j) & (ps - 1))) * D;
      attn_copy((const char*)base + koff, k_lds + (buf * ATTN_KT * KC + i * ATTN_THREADS) * 16);
    }
    const bf16_t* vp = a.v + ((((int64_t)max(pn, 0) * a.Hkv + h) * D + vrow) << a.seqs.lp) + ((t + 8 * vc) & (ps - 1));
#pragma unroll
    for (int i = 0; i < NV; ++i)
      attn_copy(vp + ((int64_t)(32 * i) << a.seqs.lp), v_lds + (buf * D * 8 + i * ATTN_THREADS) * 16);
  };
  const int low0 = attn_limit(a, w, 0);  // every row of the tile attends the tokens up to here
  const a_u4* const kb0 = &k_s[0][col * KC];
  const a_u4* const vb0 = &v_s[0][col * 8];
  const int ksw = KC == 16 ? col & 15 : (col >> 1) & 7, vsw = (col >> 1) & 7;

  int t = w.lo, buf = 0;
  if (tid < 2) bad_s[tid] = -1;
  entry(t);
  a_u4 qf[D / 16];
  const bf16_t* const src = attn_query(a, w, h, min(r, w.nr - 1)) + 8 * e;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) qf[s] = *(const a_u4*)(src + 16 * s);
  paged_asked();
  pn = page(t);
  entry(t + ATTN_KT);
  load(t, 0);
  if constexpr (EIGHT) widen(0);
#pragma unroll
  for (int s = 0; s < D / 16; ++s) qf[s] = in ? qf[s] ^ a.flip : a_mk(0, 0, 0, 0);
  f32x16_t o[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b)
#pragma unroll
    for (int q = 0; q < 16; ++q) o[b][q] = 0.0f;
  float m = ATTN_LOW, l = 0.0f;
  bool far = true;  // some row's m is beyond ATTN_FAR
  while (true) {
    attn_landed();  // the present step is in its buffer, and every wave is done with the other one
    const bool more = t + ATTN_KT < w.hi;
    // operands of the first product, two k steps at a time: the first two's are on their way before the
    // copies, the next two's before the present two's products
    const a_u4* const kb = kb0 + buf * (ATTN_KT * KC);
    a_u4 xk[2][4];
    auto get_k = [&](a_u4 (&f)[4], int q) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = kb[32 * (i & 1) * KC + ((2 * (q + (i >> 1)) + e) ^ ksw)];
    };
    get_k(xk[0], 0);
    __builtin_amdgcn_sched_barrier(0);
    pg = pn;
    pn = page(t + ATTN_KT);
    entry(t + 2 * ATTN_KT);
    if (more) load(t + ATTN_KT, buf ^ 1);
    // a step with a masked place: only the finite part of V, and a mark where there is another
    const int rt = w.at<WIN>(t);  // the step's first position
    const bool masked = rt + ATTN_KT - 1 > low0 || t + ATTN_KT > w.hi || (WIN && rt < high0) || __ballot(pg < 0);
    if (masked) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const a_u4 v = v_s[buf][i * ATTN_THREADS + tid];
        if (attn_bad(v) & 0x80008000u) {
          v_s[buf][i * ATTN_THREADS + tid] = attn_clean(v);
          bad_s[buf] = t;
        }
      }
      wg_lds_barrier();
    }
    const bool on = rt <= top && (!WIN || rt + ATTN_KT > bottom || rt < a.sinks);  // some row of the wave attends the step
    f32x16_t s[2];
    if (on) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int q = 0; q < 16; ++q) s[b][q] = 0.0f;
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int q = 0; q < D / 16; q += 2) {
        if (q + 2 < D / 16) get_k(xk[((q >> 1) + 1) & 1], q + 2);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i & 1] = mfma32a(xk[(q >> 1) & 1][i], qf[q + (i >> 1)], s[i & 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
    }
    if (on) {
      // the second product's first operands
      const a_u4* const vb = vb0 + buf * (D * 8);
      a_u4 x[2][MB], pf[2];
      auto get = [&](a_u4 (&f)[MB], int kk) {
#pragma unroll
        for (int b = 0; b < MB; ++b) f[b] = vb[32 * b * 8 + ((2 * kk + e) ^ vsw)];
      };
      get(x[0], 0);
      __builtin_amdgcn_sched_barrier(0);
      const uint64_t have = __ballot(pg >= 0);  // bit 2 j ^ of_odd: group j
      const int last = min(limit - rt, w.hi - 1 - t) - 8 * e;  // of the lane's tokens, 16 (2 b + q / 8) + q % 8
      const int first = from - rt - 8 * e, kept = a.sinks - rt - 8 * e;
      if (rt + ATTN_KT - 1 > low || t + ATTN_KT > w.hi || (WIN && rt < high) || have != ~0ull) {  // a masked place
        asm volatile("");  // a branch: few steps have one
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const int i = 16 * (2 * b + (q >> 3)) + (q & 7);
            s[b][q] = i <= last && (!WIN || i >= first || i < kept) ? s[b][q] : -__builtin_inff();
          }
        if (have != ~0ull) {  // a group without a page
          asm volatile("");
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int q = 0; q < 16; ++q)
              s[b][q] = (have >> ((2 * (2 * b + (q >> 3))) ^ of_odd)) & 1 ? s[b][q] : -__builtin_inff();
        }
      }
      float mx = ATTN_LOW;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int q = 0; q < 16; q += 2) mx = attn_max3(mx, s[b][q], s[b][q + 1]);
      mx = fmaxf(mx, pl_xor32f(mx, lane)) * a.c;
      // m follows the maximum only where it has grown by more than ATTN_SLACK: p stays below
      // 2^ATTN_SLACK, and most steps leave o and l as they are
      if (__ballot(mx > m + ATTN_SLACK)) {
        const float mn = fmaxf(m, mx), shrink = attn_exp2(m - mn);
        l *= shrink;
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
          for (int q = 0; q < 16; ++q) o[b][q] *= shrink;
        m = mn;
        far = __ballot(fabsf(m) >= ATTN_FAR) != 0;
      }
      float cw = a.c, mw = m;
      if (far) {
        asm volatile("");  // a branch: few steps have one
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int q = 0; q < 16; ++q) s[b][q] = __fmul_rn(s[b][q], a.c) - m;
        cw = 1.0f, mw = 0.0f;
      }
      // the second product, 16 tokens at a time: a product's time is that of a few of the next tokens'
      // exponentials, which stand between the products
      auto weigh = [&](int kk, int j) {  // P of tokens 2 j and 2 j + 1 of 8
        const float u = s[kk >> 1][8 * (kk & 1) + 2 * j], v = s[kk >> 1][8 * (kk & 1) + 2 * j + 1];
        const float p0 = attn_exp2(__fmaf_rn(u, cw, -mw)), p1 = attn_exp2(__fmaf_rn(v, cw, -mw));
        pf[kk & 1][j] = f32_to_bf16x2(p0, p1);
        l = attn_sum2(pf[kk & 1][j], l);
      };
#pragma unroll
      for (int j = 0; j < 4; ++j) weigh(0, j);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        if (kk < 3) get(x[(kk + 1) & 1], kk + 1);
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          __builtin_amdgcn_sched_barrier(0);
          o[b] = mfma32a(x[kk & 1][b], pf[kk & 1], o[b]);
          if (kk < 3) {
#pragma unroll
            for (int j = b * 4 / MB; j < (b + 1) * 4 / MB; ++j) weigh(kk + 1, j);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(0);
      if (masked && __builtin_amdgcn_readfirstlane(bad_s[buf]) == t) {  // what was taken out of V, read again, for the rows that attend it
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          f32x16_t code;
#pragma unroll
          for (int q = 0; q < 16; ++q) code[q] = 0.0f;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const int64_t head = (int64_t)max(__builtin_amdgcn_readlane(pg, (2 * kk) ^ of_odd), 0) * a.Hkv + h;
            const int place = (rt + 16 * kk) & (ps - 1);
            const int n = (have >> ((2 * kk) ^ of_odd)) & 1 ? min(max(last - 16 * kk + 1, 0), 8) : 0;  // attended of 8
            uint32_t seen = (1u << n) - 1;
            if constexpr (WIN) {
              const uint32_t before = (1u << min(max(first - 16 * kk, 0), 8)) - 1, stay = (1u << min(max(kept - 16 * kk, 0), 8)) - 1;
              seen &= ~before | stay;
            }
            a_u4 x;
            if constexpr (EIGHT) {
              const int64_t block = ((head << a.seqs.lp) + place) >> 4;
              const uint2 y = *(const uint2*)((const uint8_t*)a.v + (block * D + 32 * b + col) * 16 + 8 * e);
              const float f = fp8_factor(a.vs[block]);
              x = a_mk(fp8_bf16<false>(y.x, f), fp8_bf16<true>(y.x, f), fp8_bf16<false>(y.y, f), fp8_bf16<true>(y.y, f));
            } else {
              x = *(const a_u4*)(a.v + ((head * D + 32 * b + col) << a.seqs.lp) + place + 8 * e);
            }
            code = mfma32a(attn_code(x), attn_ones(seen), code);
          }
#pragma unroll
          for (int q = 0; q < 16; ++q) o[b][q] = attn_poison(o[b][q], code[q]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    if (!more) break;
    buf ^= 1;
    t += ATTN_KT;
    if constexpr (EIGHT) widen(buf);
  }

  l += pl_xor32f(l, lane);
  if (!in) return;
  const int64_t row = attn_row(a, w, h, r);
  if (w.ns == 1) {
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    bf16_t* to = a.out + row * D + 4 * e;
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(uint2*)(to + 32 * b + 8 * q) = make_uint2(f32_to_bf16x2(o[b][4 * q] * inv, o[b][4 * q + 1] * inv),
                                                    f32_to_bf16x2(o[b][4 * q + 2] * inv, o[b][4 * q + 3] * inv));
  } else {
    float* to = a.po + (row * a.splits + split) * D + 4 * e;
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(float4*)(to + 32 * b + 8 * q) = make_float4(o[b][4 * q], o[b][4 * q + 1], o[b][4 * q + 2], o[b][4 * q + 3]);
    if (e == 0) *(float2*)(a.pml + (row * a.splits + split) * 2) = make_float2(m, l);
  }
  if (a.splits > 1 && split == 0 && e == 0) a.pns[row] = w.ns;
}

// ------------------------------------------------------------------ join
// D / 4 threads per row (token and query head), four channels each. Bound by the read of the ranges'
// results, which the caches still hold (7 us for 2048 tokens of 12 heads in two ranges, 50 MB), and by its
// chain of loads when they are few (3.1 us for 12 rows of nine). With few ranges a workgroup takes
// as many rows as fit (ALONE); with many it takes one row, its groups of threads alternate ranges,
// added in order through LDS.
#define ATTN_MAX_SPLITS 64
#define ATTN_SPREAD 16  // workgroups of 16-row tiles per CU beyond which more ranges even nothing out
#define ATTN_JOIN_ALONE 8  // ranges up to which a row's threads add them alone

template <int D, bool ALONE>
__global__ __launch_bounds__(ATTN_THREADS) void attn_join_kernel(AttnArgs a, int64_t rows) {
  constexpr int T = D / 4, G = ATTN_THREADS / T;
  const int g = threadIdx.x / T, d = 4 * (threadIdx.x % T);
  const int64_t row = ALONE ? (int64_t)blockIdx.x * G + g : blockIdx.x;
  const int ns = row < rows ? min(a.pns[row], a.splits) : 0;
  if (ns <= 1) return;  // written already (ALONE: no barrier follows; otherwise one row, one answer)
  const float2* const ml = (const float2*)a.pml + row * a.splits;
  const float* const from = a.po + row * a.splits * D + d;
  float m = ATTN_LOW;
  for (int i = 0; i < ns; ++i) m = fmaxf(m, ml[i].x);
  float l = 0.0f;
  f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int i = ALONE ? 0 : g; i < ns; i += ALONE ? 1 : G) {
    const float2 x = ml[i];
    const float f = attn_exp2(x.x - m);
    const f32x4_t p = *(const f32x4_t*)(from + (int64_t)i * D);
    l = __fmaf_rn(x.y, f, l);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = __fmaf_rn(p[j], f, acc[j]);
  }
  if (!ALONE) {
    __shared__ f32x4_t acc_s[G][T];
    __shared__ float l_s[G];
    acc_s[g][d / 4] = acc;
    if (d == 0) l_s[g] = l;
    __syncthreads();
    if (g) return;
    for (int i = 1; i < G; ++i) {
      acc += acc_s[i][d / 4];
      l += l_s[i];
    }
  }
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  *(uint2*)(a.out + row * D + d) = make_uint2(f32_to_bf16x2(acc[0] * inv, acc[1] * inv), f32_to_bf16x2(acc[2] * inv, acc[3] * inv));
}

// ------------------------------------------------------------------ host
struct AttnPlan {
  int rows;    // per tile: 16 or ATTN_ROWS
  int splits, base, behind;
  int64_t tiles;
};

// (window and sinks: what a tile's steps hold of them at most, as though the table were no longer)
static AttnPlan attn_plan(int64_t n_tokens, int n_seqs, int max_pages, int page_size, int Hq, int Hkv, int D, int64_t window,
                          int64_t sinks) {
  AttnPlan p = {};
  const int64_t rows = n_tokens * (Hq / Hkv), cus = pp_device_cus(), room = (int64_t)max_pages * page_size;
  const int64_t capacity = window > 0 ? std::min(room, std::min(window, room) + std::min(sinks, room) + 2 * ATTN_ROWS) : room;
  auto items = [&](int tile) { return std::max<int64_t>(1, (rows / tile + n_seqs) * Hkv); };
  // Tiles of 16 rows for single tokens and the like, for what does not fill the GPU, and for what is short
  // altogether: their steps cost four times as much for the same work (6 ns for 16 rows x 128 tokens of D = 128,
  // the whole GPU at work, against 1.4), but there are eight times as many tiles. 12 heads: prompts of 200, 512,
  // 700 and 1024 tokens 6.9, 12.3, 16.7 and 25.0 us, tiles of 128 rows 10.8, 17.5, 21.2 and 23.3; 128 new tokens
  // at 8000 51 against 32. Sequences of one length, 64 of up to 8000 tokens: 1, 4, 8, 16 rows each 423, 422, 439,
  // 470 us, tiles of 128 rows 468, 452, 462, 455; 32 heads on 8, 4, 8, 16 rows 298, 305, 406 against 292, 295,
  // 298; one of 8000, 8 rows, 11.5 against 19.0. Up to 4 rows a sequence, as a mean, so that a chunk among
  // single tokens does not come to tiles of 16 rows, which is what the step of a server has: 63 single tokens and
  // 900 at 8000 362 us, in tiles of 128 rows 229; 255 and 3800 at 4000 953 and 449 (32 heads on 8 1756 and 577).
  const bool few = rows <= 4 * (int64_t)n_seqs || (rows <= 16 * (int64_t)n_seqs && items(16) <= cus) ||
                   items(16) * ((capacity + 127) / 128) <= 4096;
  p.rows = few ? 16 : ATTN_ROWS;
  p.tiles = rows / p.rows + n_seqs + 1;
  const int64_t each = items(p.rows);
  int64_t most;
  if (few) {
    // As many ranges as give every CU one, and at least one per 1024 tokens, so that sequences of different
    // lengths even out. 12 heads, one token: 256, 512, 1024, 2048, 4096 tokens 7.0, 9.2, 13.5, 22.3, 40.6 us, in
    // ranges of 128 8.1, 8.2, 8.8, 9.4, 12.1; 16 sequences of 1024 19.2, in 6 ranges 22.9; 64 of 1 to 8192 tokens
    // in 1, 2, 8 ranges 343, 300, 271. The width of the table and ATTN_SPREAD workgroups a CU bound them, and so
    // the grid and the workspace: for 8, 16, 32 a CU 64 sequences of 1 to 8192 tokens 292, 283, 280 us, 64 of 500
    // in a table of 32000 tokens 36, 42, 51 (33 in one of 512; by the width alone 192); the workspace stays below
    // that many workgroups' 16 rows of D + 2 floats, 35 MB, and one more range of every row.
    p.base = (int)std::max<int64_t>(1, cus / each);
    most = capacity <= 384 ? 1 : std::max<int64_t>(p.base, std::min(capacity / 1024, (ATTN_SPREAD * cus + each - 1) / each));
    most = std::min(most, (capacity + 127) / 128);
  } else {
    // One round of the workgroups that the GPU holds (2 per CU at D = 128, 3 at D = 64): a part of a round more
    // is a round of its own where all tiles are about as long, in a chunk of one sequence far behind the
    // cache's start (`behind`: as long again and more before it). Those of a prompt and of several sequences
    // differ, and there a part of a round does no harm while there are few ranges.
    // us for 1, 2, 3, 4 ranges: prompts of 2048 tokens (204 items) 49, 42, 37, 45; of 4096 (396) 97, 86, 93,
    // 103; of 8192 (780) 231, and 265 with even one tile cut; new tokens at 8000: 1500 (144) 196, 135, 113,
    // 133, 2048 208, 154, 174, 150, 4096 306, 318, 331, 319; for 6, 8, 10: 512 new at 30000 (60) 157, 137,
    // 126, of D = 64 (500 at 29511, 128 items) 165, 184, 194;
    // for 1, 2: nine sequences of 700 new tokens at 4000 and single ones 116, 86.
    const int64_t slots = (D == 64 ? 3 : 2) * cus;
    p.behind = (int)std::max<int64_t>(1, slots / each);
    // Tiles of a window are as long as each other: a part of a round more is one of its own there too. A window of 1024, 12
    // heads, prompts of 3000, 4096, 5000 tokens 41, 51, 52 us, with the part of a round (two ranges) 51, 64, 75; of 8192
    // (1.5 rounds) 88, the half of a round in two ranges 92.
    p.base = p.behind >= 4 || window > 0 ? p.behind : (int)((slots + each - 1) / each);
    most = std::min<int64_t>(p.base, (capacity + 511) / 512);
  }
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(ATTN_MAX_SPLITS, most));
  return p;
}

static size_t attn_ws_bytes(const AttnPlan& p, int64_t rows, int D) {
  if (p.splits == 1) return 0;
  return (size_t)rows * p.splits * (D + 2) * 4 + (size_t)rows * 4;
}

static int attn_window(const char* what, int64_t window, int64_t sinks) {
  PP_REQUIRE(window >= 0 && sinks >= 0, PP_ERR_INVALID, "%s: window %lld, %lld first tokens", what, (long long)window, (long long)sinks);
  return PP_OK;
}

extern "C" size_t pp_paged_attention_with_workspace_bytes(int64_t n_tokens, int n_seqs, int max_pages, int page_size, int Hq, int Hkv,
                                                          int D, int eight_bits, int64_t window, int64_t sinks) {
  const char* const what = "pp_paged_attention";
  if (pp_paged_sizes(what, n_tokens, n_seqs, max_pages, 1, page_size, Hq, Hkv, D) || attn_window(what, window, sinks)) return 0;
  if (n_tokens == 0 || Hq == 0) return 0;
  return attn_ws_bytes(attn_plan(n_tokens, n_seqs, max_pages, page_size, Hq, Hkv, D, window, sinks), n_tokens * Hq, D);
}

extern "C" size_t pp_paged_attention_workspace_bytes(int64_t n_tokens, int n_seqs, int max_pages, int page_size,
                                                     int Hq, int Hkv, int D) {
  return pp_paged_attention_with_workspace_bytes(n_tokens, n_seqs, max_pages, page_size, Hq, Hkv, D, 0, 0, 0);
}

static int attend(const char* what, const void* q, const int64_t* q_strides, int64_t n_tokens, int n_seqs, const int32_t* cu_q,
                  const int32_t* kv_lens, const int32_t* block_table, int max_pages, const void* k_pages, const void* v_pages,
                  const void* k_scales, const void* v_scales, int num_pages, int page_size, int Hq, int Hkv, int D, float scale,
                  int64_t window, int64_t sinks, void* out_bf16, int zero_tail, void* workspace, size_t workspace_bytes,
                  void* stream) {
  int rc = pp_paged_check(what, n_tokens, n_seqs, cu_q, kv_lens, block_table, max_pages, k_pages, v_pages, num_pages,
                          page_size, Hq, Hkv, D);
  if (rc) return rc;
  PP_REQUIRE(Hq >= 1, PP_ERR_INVALID, "%s: no query heads", what);
  PP_REQUIRE(!k_scales == !v_scales, PP_ERR_INVALID, "%s: scales of keys and of values belong together", what);
  rc = attn_window(what, window, sinks);
  if (rc) return rc;
  if (n_tokens == 0) return PP_OK;
  PP_REQUIRE(q && q_strides && out_bf16, PP_ERR_INVALID, "%s: null pointer", what);
  PP_REQUIRE((((uintptr_t)q | (uintptr_t)out_bf16) & 15) == 0 && q_strides[0] % 8 == 0 && q_strides[1] % 8 == 0,
             PP_ERR_INVALID, "%s: every head of q and out must start on a 16-byte boundary", what);
  const float c = fabsf(scale) * 1.4426950408889634f;
  PP_REQUIRE(std::isfinite(c), PP_ERR_INVALID, "%s: scale %g", what, scale);
  const AttnPlan p = attn_plan(n_tokens, n_seqs, max_pages, page_size, Hq, Hkv, D, window, sinks);
  const size_t need = attn_ws_bytes(p, n_tokens * Hq, D);
  PP_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), PP_ERR_INVALID,
             "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", what, workspace_bytes, need);
  AttnArgs a;
  a.seqs = {cu_q, kv_lens, block_table, (int)n_tokens, n_seqs, max_pages, num_pages, paged_log2(page_size)};
  a.q = (const bf16_t*)q, a.qs[0] = q_strides[0], a.qs[1] = q_strides[1];
  a.k = (const bf16_t*)k_pages, a.v = (const bf16_t*)v_pages;
  a.Hq = Hq, a.Hkv = Hkv, a.group = Hq / Hkv;
  a.c = std::max(c, 0x1p-149f), a.flip = scale < 0.0f ? 0x80008000u : 0u;  // (for 0: 2^-21 of any float32)
  a.out = (bf16_t*)out_bf16, a.zero_tail = zero_tail;
  a.splits = p.splits, a.base = p.base, a.behind = p.behind, a.tiles = (int)p.tiles;
  a.ks = (const uint8_t*)k_scales, a.vs = (const uint8_t*)v_scales;
  // (no position is beyond 2^31, none in the table beyond 2^30)
  a.window = (int)std::min<int64_t>(window, 0x7fffffff), a.sinks = (int)std::min<int64_t>(sinks, 1 << 30);
  a.po = (float*)workspace;
  a.pml = a.po + n_tokens * Hq * p.splits * D;
  a.pns = (int*)(a.pml + n_tokens * Hq * p.splits * 2);
  const int64_t items = p.tiles * Hkv * p.splits, rows = n_tokens * Hq;
  const bool alone = p.splits <= ATTN_JOIN_ALONE;
  // (the join's are never more: eight rows each and more where there are few ranges, which is two workgroups to a
  // tile of 16 rows; calls of more than 8 ranges, and cut tiles of 128 rows, are no more than the GPU holds some
  // times over)
  // The limit goes by the shapes alone, not by the GPU's size or the tile: up to 16 rows a sequence it counts tiles
  // of 16 rows with a range per 1024 tokens of the table (64 at most), which a launch never has.
  const int64_t per_head = n_tokens * a.group, ranges = std::min<int64_t>(ATTN_MAX_SPLITS, (int64_t)max_pages * page_size / 1024);
  const int64_t counted = std::max(items, per_head <= 16 * (int64_t)n_seqs ? (per_head / 16 + n_seqs + 1) * Hkv * ranges : 0);
  PP_REQUIRE(counted <= 0xffffff, PP_ERR_UNSUPPORTED, "%s: %lld workgroups (at most 2^24 - 1)", what, (long long)counted);
  const int64_t joins = alone ? (rows * (D / 4) + ATTN_THREADS - 1) / ATTN_THREADS : rows;
  hipStream_t st = (hipStream_t)stream;
  const unsigned n = (unsigned)items, nj = (unsigned)joins;
#define ATTN_KIND(D_, EIGHT_, WIN_)                                                       \
  do {                                                                                    \
    if (p.rows == 16) attn_few_kernel<D_, EIGHT_, WIN_><<<n, ATTN_THREADS, 0, st>>>(a);   \
    else attn_many_kernel<D_, EIGHT_, WIN_><<<n, ATTN_THREADS, 0, st>>>(a);               \
  } while (0)
#define ATTN(D_)                                                                          \
  do {                                                                                    \
    if (k_scales && window > 0) ATTN_KIND(D_, true, true);                                \
    else if (k_scales) ATTN_KIND(D_, true, false);                                        \
    else if (window > 0) ATTN_KIND(D_, false, true);                                      \
    else ATTN_KIND(D_, false, false);                                                     \
    if (p.splits > 1) {                                                                   \
      if (alone) attn_join_kernel<D_, true><<<nj, ATTN_THREADS, 0, st>>>(a, rows);        \
      else attn_join_kernel<D_, false><<<nj, ATTN_THREADS, 0, st>>>(a, rows);             \
    }                                                                                     \
  } while (0)
  if (D == 64) ATTN(64);
  else ATTN(128);
#undef ATTN
#undef ATTN_KIND
  return pp_check_launch(what);
}

extern "C" int pp_paged_attention(const void* q, const int64_t* q_strides, int64_t n_tokens, int n_seqs,
                                  const int32_t* cu_q, const int32_t* kv_lens, const int32_t* block_table,
                                  int max_pages, const void* k_pages, const void* v_pages, int num_pages,
                                  int page_size, int Hq, int Hkv, int D, float scale, void* out_bf16, int zero_tail,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  return attend("pp_paged_attention", q, q_strides, n_tokens, n_seqs, cu_q, kv_lens, block_table, max_pages, k_pages, v_pages,
                nullptr, nullptr, num_pages, page_size, Hq, Hkv, D, scale, 0, 0, out_bf16, zero_tail, workspace,
                workspace_bytes, stream);
}

extern "C" int pp_paged_attention_with(const void* q, const int64_t* q_strides, int64_t n_tokens, int n_seqs, const int32_t* cu_q,
                                       const int32_t* kv_lens, const int32_t* block_table, int max_pages, const void* k_pages,
                                       const void* v_pages, const void* k_scales, const void* v_scales, int num_pages,
                                       int page_size, int Hq, int Hkv, int D, float scale, int64_t window, int64_t sinks,
                                       void* out_bf16, int zero_tail, void* workspace, size_t workspace_bytes, void* stream) {
  return attend("pp_paged_attention_with", q, q_strides, n_tokens, n_seqs, cu_q, kv_lens, block_table, max_pages, k_pages,
                v_pages, k_scales, v_scales, num_pages, page_size, Hq, Hkv, D, scale, window, sinks, out_bf16, zero_tail,
                workspace, workspace_bytes, stream);
}
