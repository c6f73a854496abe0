// Shared device pieces of the attention with a bucketed relative position bias (rel_attn.hip, rel_attn_bwd.hip).
//
// Both directions are written on 32 x 32 score tiles of v_mfma_f32_32x32x16_bf16 in the orientation that keeps the
// scores in registers: the accumulator of one product is the B operand of the next.  A lane holds ONE column of the tile
// (lane & 31) and 16 of its 32 rows, row(r) = (r & 3) + 8 (r >> 2) + 4 (lane >> 5); registers 0..7 are then a B operand of
// 16 k-values {4 lk + 0..3, 8 + 4 lk + 0..3}, registers 8..15 the next 16.  The A operand of that second product is read
// from a TRANSPOSED image of the tile whose 4-row groups are stored in the same order (ra_store_trans).
//
// Products: bf16 inputs are one product.  fp32 inputs are split into three bf16 pieces (x = h + m + l, 24 bits) and a
// product is the six terms above 2^-24; the two-piece, three-term form the other attention kernels use leaves 3e-6 ... 5e-6
// of error, which the position bias' gradient (sums with cancellation) would show.
#pragma once
#include "occf_common.h"

#define RA_LOG2E 1.44269504088896340736f
#define RA_PAD 64               // bias columns kept beyond either end of the clamped distances

#ifdef OCCF_EMU
#define ra_mfma16(a, b, c) emu_mfma_f32_16x16x32_bf16(a, b, c)
#define RA_WAVE_SYNC() hipemu::wave_sync()
static inline float ra_exp2(float x) { return exp2f(x); }
static inline float ra_log2(float x) { return log2f(x); }
#else
typedef __bf16 ra_bf16x8 __attribute__((ext_vector_type(8)));
#define ra_mfma16(a, b, c) \
  __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ra_bf16x8, a), __builtin_bit_cast(ra_bf16x8, b), c, 0, 0, 0)
// a wave's own LDS writes become visible to its other lanes (LDS operations of one wave complete in order)
#define RA_WAVE_SYNC()                                    \
  do {                                                    \
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront"); \
    __builtin_amdgcn_wave_barrier();                      \
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront"); \
  } while (0)
__device__ __forceinline__ float ra_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float ra_log2(float x) { return __builtin_amdgcn_logf(x); }
#endif

typedef uint16_t ra_bf16;
template <class T> struct RaType;
template <> struct RaType<float> { static constexpr int NT = 3; };
template <> struct RaType<ra_bf16> { static constexpr int NT = 1; };

// waves a SIMD that the backward kernels are compiled for: two where their accumulators, fixed operands and tiles in flight fit
// 256 registers, else one with 512
#define RA_WAVES_PER_SIMD(T, DP) (DP <= (RaType<T>::NT == 3 ? 32 : 64) ? 2 : 1)

struct RaParams {
  const void *q, *k, *v, *table, *out, *dout;
  const int32_t *lut, *q_lens, *k_lens, *q_start;
  void *o, *dq, *dk, *dv;
  float *lse, *delta, *part;
  long qsb, qsl, qsh, ksb, ksl, ksh, vsb, vsl, vsh;     // element strides: batch, row, head
  int B, Lq, Lk, Hq, Hk, D, nb, R, causal, nsplit, chunk, units, by_length;
  float scale, c;                                          // c = scale * log2(e)
};

template <int NT> struct RaFrag { bf16x8 p[NT]; };

template <int NT>
__device__ __forceinline__ f32x16 ra_mm(const RaFrag<NT>& a, const RaFrag<NT>& b, f32x16 c) {
  if constexpr (NT == 3) {
    c = occf_mfma_bf16_32x32x16(a.p[2], b.p[0], c);
    c = occf_mfma_bf16_32x32x16(a.p[0], b.p[2], c);
    c = occf_mfma_bf16_32x32x16(a.p[1], b.p[1], c);
    c = occf_mfma_bf16_32x32x16(a.p[1], b.p[0], c);
    c = occf_mfma_bf16_32x32x16(a.p[0], b.p[1], c);
  }
  return occf_mfma_bf16_32x32x16(a.p[0], b.p[0], c);
}

__device__ __forceinline__ f32x16 ra_zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

// two values -> NT packed bf16 pairs
template <int NT>
__device__ __forceinline__ void ra_split2(float a, float b, uint32_t (&w)[NT]) {
  w[0] = occf_bf16_pack2(a, b);
  if constexpr (NT == 3) {
    a -= occf_u2f(w[0] << 16);
    b -= occf_u2f(w[0] & 0xFFFF0000u);
    w[1] = occf_bf16_pack2(a, b);
    a -= occf_u2f(w[1] << 16);
    b -= occf_u2f(w[1] & 0xFFFF0000u);
    w[2] = occf_bf16_pack2(a, b);
  }
}

struct RaU4 { uint32_t x[4]; };
__device__ __forceinline__ bf16x8 ra_as_frag(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const RaU4 u = {{a, b, c, d}};
#ifdef OCCF_EMU
  bf16x8 f;
  memcpy(&f, &u, 16);
  return f;
#else
  return __builtin_bit_cast(bf16x8, u);
#endif
}

// eight consecutive register values -> B operand
template <int NT>
__device__ __forceinline__ RaFrag<NT> ra_pack8(const float* v) {
  uint32_t w[4][NT];
#pragma unroll
  for (int e = 0; e < 4; ++e) ra_split2<NT>(v[2 * e], v[2 * e + 1], w[e]);
  RaFrag<NT> f;
#pragma unroll
  for (int t = 0; t < NT; ++t) f.p[t] = ra_as_frag(w[0][t], w[1][t], w[2][t], w[3][t]);
  return f;
}

// 8 consecutive elements of a row (16-byte aligned; `ok` false gives zeros) -> fragment
template <class T>
__device__ __forceinline__ RaFrag<RaType<T>::NT> ra_row_frag(const T* p, bool ok) {
  if constexpr (RaType<T>::NT == 1) {
    RaU4 u = {{0u, 0u, 0u, 0u}};
    if (ok) u = *(const RaU4*)__builtin_assume_aligned(p, 16);
    RaFrag<1> f;
    f.p[0] = ra_as_frag(u.x[0], u.x[1], u.x[2], u.x[3]);
    return f;
  } else {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 0.f;
    if (ok) {
      const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
      f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
    return ra_pack8<3>(f);
  }
}

__device__ __forceinline__ float ra_to_float(float x) { return x; }
__device__ __forceinline__ float ra_to_float(ra_bf16 x) { return occf_u2f((uint32_t)x << 16); }

__device__ __forceinline__ void ra_store4(float* p, float a, float b, float c, float d) {
  *(float4*)p = make_float4(a, b, c, d);
}
__device__ __forceinline__ void ra_store4(ra_bf16* p, float a, float b, float c, float d) {
  struct U2 { uint32_t x, y; };
  *(U2*)__builtin_assume_aligned(p, 8) = U2{occf_bf16_pack2(a, b), occf_bf16_pack2(c, d)};
}

// LDS images of a tile of ROWS x DP, one per piece.
//   row image:   [ROWS][DP], 16 bytes of padding a row: the 16-lane groups of a b128 read hit 16 different bank quads
//   trans image: [DP][ROWS], 4-row groups in operand order, 16 bytes of padding, the 16-byte slots of a row exchanged by
//                (column >> 4) & 3 so that the 16 column groups of a store do not meet on one bank quad
template <int DP> struct RaRow {
  static constexpr int LD = DP * 2 + 16;
  static constexpr int bytes(int rows) { return rows * LD; }
};
template <int ROWS> struct RaTrans {
  static constexpr int LD = ROWS * 2 + 16;
  static constexpr int bytes(int dp) { return dp * LD; }
};

typedef uint32_t ra_u2 __attribute__((ext_vector_type(2)));

// ---- a 4 x 4 block of a tile: 4 rows x 4 columns on their way from global memory to the LDS images
template <class T> struct RaBlk;

// bounded loads (no branch a load: under branches every load is waited for where the paths meet).  The resource starts at the tile's first row, so that 32-bit offsets reach it wherever it lies; a tile's rows
// span less than 2 GiB (ra_check)
#ifdef OCCF_EMU
static inline RaU4 ra_buf16(occf_bbuf b, uint32_t off) {
  const occf_u32x4 v = occf_bbuf_load_b128(b, off);
  return RaU4{{v.x, v.y, v.z, v.w}};
}
struct ra_raw2 { uint32_t x, y; };
static inline ra_raw2 ra_buf8(occf_bbuf b, uint32_t off) {
  ra_raw2 v = {0u, 0u};
  if ((uint64_t)off + 8u <= (uint64_t)b.nbytes) memcpy(&v, b.base + off, 8);
  return v;
}
#else
__device__ __forceinline__ RaU4 ra_buf16(occf_bbuf b, uint32_t off) {
  return __builtin_bit_cast(RaU4, __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, 0));
}
struct ra_raw2 { uint32_t x, y; };
__device__ __forceinline__ ra_raw2 ra_buf8(occf_bbuf b, uint32_t off) {
  return __builtin_bit_cast(ra_raw2, __builtin_amdgcn_raw_buffer_load_b64(b, off, 0, 0));
}
#endif
template <> struct RaBlk<float> { RaU4 r[4]; };
template <> struct RaBlk<ra_bf16> { ra_raw2 r[4]; };

// the next `rows` rows from `tile`: the resource ends with the last of them (rows lie D or more apart, ra_check), so that the
// rows behind read as zeros without a test
template <class T>
__device__ __forceinline__ occf_bbuf ra_tile(const T* tile, long stride, int rows, int D) {
  const int n = rows < 64 ? rows : 64;
  return occf_make_bbuf(tile, n > 0 ? ((uint32_t)(n - 1) * (uint32_t)stride + (uint32_t)D) * (uint32_t)sizeof(T) : 0u);
}

// byte offset of block u of a tile (u = row group * (DP / 4) + column group); columns at or behind D lie outside any tile
template <class T, int DP>
__device__ __forceinline__ uint32_t ra_blk_at(long stride, int D, int u) {
  const int c = (u % (DP / 4)) * 4, r0 = (u / (DP / 4)) * 4;
  return c < D ? ((uint32_t)r0 * (uint32_t)stride + (uint32_t)c) * (uint32_t)sizeof(T) : OCCF_BUF_OOB;
}
template <class T>
__device__ __forceinline__ void ra_load_blk(RaBlk<T>& b, occf_bbuf buf, uint32_t at, long stride) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t off = at + i * ((uint32_t)stride * (uint32_t)sizeof(T));
    if constexpr (sizeof(T) == 4) b.r[i] = ra_buf16(buf, off);
    else b.r[i] = ra_buf8(buf, off);
  }
}

// 8 columns from `c` of row `row` of such a tile, as loaded and as a fragment
template <class T> struct RaRaw { RaU4 x[sizeof(T) / 2]; };
template <class T>
__device__ __forceinline__ uint32_t ra_raw_at(long stride, int D, int row, int c) {
  return c < D ? ((uint32_t)row * (uint32_t)stride + (uint32_t)c) * (uint32_t)sizeof(T) : OCCF_BUF_OOB;
}
template <class T>
__device__ __forceinline__ void ra_load_raw(RaRaw<T>& f, occf_bbuf buf, uint32_t at) {
#pragma unroll
  for (int e = 0; e < (int)sizeof(T) / 2; ++e) f.x[e] = ra_buf16(buf, at + 16u * e);
}
__device__ __forceinline__ RaFrag<1> ra_raw_frag(const RaRaw<ra_bf16>& w) {
  RaFrag<1> f;
  f.p[0] = ra_as_frag(w.x[0].x[0], w.x[0].x[1], w.x[0].x[2], w.x[0].x[3]);
  return f;
}
__device__ __forceinline__ RaFrag<3> ra_raw_frag(const RaRaw<float>& w) {
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = occf_u2f(w.x[e >> 2].x[e & 3]);
  return ra_pack8<3>(f);
}

// block -> packed pieces, w[piece][row][pair of columns]
__device__ __forceinline__ void ra_blk_pieces(const RaBlk<ra_bf16>& b, uint32_t (&w)[1][4][2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[0][i][0] = b.r[i].x;
    w[0][i][1] = b.r[i].y;
  }
}
__device__ __forceinline__ void ra_blk_pieces(const RaBlk<float>& b, uint32_t (&w)[3][4][2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t s[3];
    ra_split2<3>(occf_u2f(b.r[i].x[0]), occf_u2f(b.r[i].x[1]), s);
#pragma unroll
    for (int t = 0; t < 3; ++t) w[t][i][0] = s[t];
    ra_split2<3>(occf_u2f(b.r[i].x[2]), occf_u2f(b.r[i].x[3]), s);
#pragma unroll
    for (int t = 0; t < 3; ++t) w[t][i][1] = s[t];
  }
}


template <int NT, int DP, int ROWS>
__device__ __forceinline__ void ra_store_row(char* img, const uint32_t (&w)[NT][4][2], int u) {
  const int c = (u % (DP / 4)) * 4, rg = u / (DP / 4);
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const ra_u2 x = {w[t][i][0], w[t][i][1]};
      *(ra_u2*)(img + t * RaRow<DP>::bytes(ROWS) + (rg * 4 + i) * RaRow<DP>::LD + c * 2) = x;
    }
}

// the low (or high) halves of two words side by side
__device__ __forceinline__ uint32_t ra_halves(uint32_t a, uint32_t b, int high) {
#ifdef OCCF_EMU
  return high ? (a >> 16) | (b & 0xFFFF0000u) : (a & 0xFFFFu) | (b << 16);
#else
  return __builtin_amdgcn_perm(b, a, high ? 0x07060302u : 0x05040100u);
#endif
}

template <int NT, int DP, int ROWS, int COLS = 32>
__device__ __forceinline__ void ra_store_trans(char* img, const uint32_t (&w)[NT][4][2], int u) {
  const int c = (u % (DP / 4)) * 4, rg = u / (DP / 4);
  // row group g of a 16-row step holds k values lk = g & 1, e = 4 (g >> 1) ..: 8-byte slot 2 lk + (g >> 1)
  const int g = rg & 3, slot = COLS == 16 ? g : (rg >> 2) * 2 + (g & 1), half = COLS == 16 ? rg >> 2 : g >> 1;
  const int off = ((slot ^ ((c >> 4) & 3)) * 16) + half * 8;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int h = j >> 1;
      const uint32_t lo = ra_halves(w[t][0][h], w[t][1][h], j & 1), hi = ra_halves(w[t][2][h], w[t][3][h], j & 1);
      const ra_u2 x = {lo, hi};
      *(ra_u2*)(img + t * RaTrans<ROWS>::bytes(DP) + (c + j) * RaTrans<ROWS>::LD + off) = x;
    }
}

// A operand: 32 rows from row0, k step ks of 16 columns
template <int NT, int DP, int ROWS>
__device__ __forceinline__ RaFrag<NT> ra_read_row(const char* img, int row0, int ks, int li, int lk) {
  RaFrag<NT> f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
    f.p[t] = *(const bf16x8*)(img + t * RaRow<DP>::bytes(ROWS) + (row0 + li) * RaRow<DP>::LD + ks * 32 + lk * 16);
  return f;
}
// A operand of the 16-column form: 16 columns of the tile from c0, its 32 rows; g = lane >> 4
template <int NT, int DP>
__device__ __forceinline__ RaFrag<NT> ra_read_trans16(const char* img, int c0, int li, int g) {
  RaFrag<NT> f;
  const int d = c0 + li;
#pragma unroll
  for (int t = 0; t < NT; ++t)
    f.p[t] = *(const bf16x8*)(img + t * RaTrans<32>::bytes(DP) + d * RaTrans<32>::LD + ((g ^ ((d >> 4) & 3)) * 16));
  return f;
}
// A operand: 32 columns of the tile from c0, k step ks of 16 tile rows
template <int NT, int DP, int ROWS>
__device__ __forceinline__ RaFrag<NT> ra_read_trans(const char* img, int c0, int ks, int li, int lk) {
  RaFrag<NT> f;
  const int d = c0 + li;
#pragma unroll
  for (int t = 0; t < NT; ++t)
    f.p[t] = *(const bf16x8*)(img + t * RaTrans<ROWS>::bytes(DP) + d * RaTrans<ROWS>::LD +
                              (((ks * 2 + lk) ^ ((d >> 4) & 3)) * 16));
  return f;
}

// ---- the same chain on 16 columns (v_mfma_f32_16x16x32_bf16): a lane holds column lane & 15 and, of 32 tile rows in two
// accumulators, rows 16 (e >> 2) + 4 (lane >> 4) + (e & 3), e = 0..7, which are one B operand of 32 k-values; the transposed
// image keeps row group g = row >> 2 at 16-byte slot g & 3, half g >> 2.
template <int NT>
__device__ __forceinline__ f32x4 ra_mm16(const RaFrag<NT>& a, const RaFrag<NT>& b, f32x4 c) {
  if constexpr (NT == 3) {
    c = ra_mfma16(a.p[2], b.p[0], c);
    c = ra_mfma16(a.p[0], b.p[2], c);
    c = ra_mfma16(a.p[1], b.p[1], c);
    c = ra_mfma16(a.p[1], b.p[0], c);
    c = ra_mfma16(a.p[0], b.p[1], c);
  }
  return ra_mfma16(a.p[0], b.p[0], c);
}

// a table entry in the base-2 domain; entries at or under -1e30 take their bucket out
__device__ __forceinline__ float ra_bias(float x) { return x <= -1e30f ? -INFINITY : x * RA_LOG2E; }

// bias of head h at every clamped distance -R .. R and RA_PAD columns of the end values on either side, base 2
template <class T>
__device__ __forceinline__ void ra_fill_bias(float* lut, const RaParams& p, int h, int tid, int nthr) {
  const T* table = (const T*)p.table;
  const int n = 2 * p.R + 1 + 2 * RA_PAD;
  for (int i = tid; i < n; i += nthr) {
    const int d = occf_clampi(i - RA_PAD, 2 * p.R);
    const int b = occf_clampi(p.lut[d], p.nb - 1);
    lut[i] = ra_bias(ra_to_float(table[(long)b * p.Hq + h]));
  }
}

// Bias and mask of a lane's 16 raw scores s, in place.  The biased base-2 score of entry r is then fma(s[r], ce, be): a tile
// further than R from the diagonal keeps its raw products (ce = c, be = the outermost bucket's bias), one near it gets the
// bias added here (ce = 1, be = 0).  `bl`: the bias of entry 0, STEP the sign of the distance along the 16 rows
// (rows = keys: +1, rows = queries: -1).  The conditions are wave-uniform; the whole tile is one branch each.
template <int STEP, class Hide>
__device__ __forceinline__ void ra_bias_mask(f32x16& s, const float* bl, bool near, float far, bool mask, float c, float& ce,
                                             float& be, Hide hide) {
  ce = c;
  be = far;
  if (near) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c, bl[STEP * ((r & 3) + 8 * (r >> 2))]);
    ce = 1.f;
    be = 0.f;
  }
  if (mask) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = hide((r & 3) + 8 * (r >> 2)) ? -INFINITY : s[r];
  }
}

__device__ __forceinline__ f32x16 ra_splat16(float x) {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = x;
  return z;
}

// Workgroup -> (tile, head of the batch).  Tiles of a head, and heads from tile to tile, go round the XCDs (workgroup n runs on
// XCD n mod 8), so that sequences of differing length spread over all of them; a head's workgroups walk its keys side by side and
// find them in their L2.  (Whole heads to an XCD leave some with the short sequences: 92 ... 157 instead of 67 us at 4 x 2500 fp32
// tokens of 0 ... 2500.)  Causal tiles differ in length: of 64 heads at a time the longest (`t` = 0) go first, so that short ones
// fill the gaps at the end; heads keep to their XCDs there unless a sequence has fewer than eight of them.
__device__ __forceinline__ void ra_order(const RaParams& p, unsigned bid, unsigned ntile, unsigned heads, int& t, int& bh) {
  if (!p.causal) {
    t = (int)(bid % ntile);
    bh = (int)(bid / ntile);
    return;
  }
  const unsigned chunk = bid / (64 * ntile), in = bid - chunk * 64 * ntile;
  const unsigned n = heads - chunk * 64 < 64 ? heads - chunk * 64 : 64;
  t = (int)(in / n);
  bh = (int)(chunk * 64 + (in + (heads < 8u * p.B ? t : 0)) % n);
}

// rows of sequence b that count: queries [0, nq), keys [0, nk), position of query 0
__device__ __forceinline__ void ra_lengths(const RaParams& p, int b, int& nq, int& nk, int& start) {
  nq = p.q_lens ? occf_clampi(p.q_lens[b], p.Lq) : p.Lq;
  nk = p.k_lens ? occf_clampi(p.k_lens[b], p.Lk) : p.Lk;
  start = p.q_start ? p.q_start[b] : 0;
  start = start < -(1 << 29) ? -(1 << 29) : (start > (1 << 29) ? (1 << 29) : start);      // distances fit 32 bits
}

// ---- host side
// geom (include/occformer_hip.h): B, Lq, Lk, Hq, Hk, D, buckets, R, strides of q, k, v
static int ra_check(const int64_t* g, int dtype) {
  if (!g || (dtype != 0 && dtype != 1)) return OCCF_EINVAL;
  const long B = g[0], Lq = g[1], Lk = g[2], Hq = g[3], Hk = g[4], D = g[5], nb = g[6], R = g[7];
  if (B <= 0 || Lq <= 0 || Lk <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || D < 8 || D > 128 || D % 8) return OCCF_ESHAPE;
  if (nb < 1 || nb > 128 || R < 1 || R > 512) return OCCF_ESHAPE;
  if (Lk > (1L << 29) || Lq > (1L << 29) || B * Hq * ((Lq + 31) / 32) * 16 >= 2147483647L ||
      B * Hk * ((Lk + 127) / 128) * 16 >= 2147483647L)
    return OCCF_ESHAPE;
  if (Lq * (Hq / Hk) >= (1L << 30) || B * Hk * ((Lq * (Hq / Hk) + 31) / 32) * 64 >= 2147483647L) return OCCF_ESHAPE;
  const long per16 = dtype == 0 ? 4 : 8;
  for (int s = 8; s < 17; ++s)
    if (g[s] < 0 || g[s] % per16) return OCCF_ESHAPE;
  for (int s = 9; s < 17; s += 3)
    if (g[s] < D || g[s] >= (1L << 22)) return OCCF_ESHAPE;      // rows apart, 64 of them within 2 GiB
  return 0;
}

template <class K, class P>
static int ra_launch(K kernel, dim3 grid, int threads, size_t lds, void* stream, const P& p) {
  if (lds > 160 * 1024) return OCCF_ESHAPE;
#ifndef OCCF_EMU
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != hipSuccess) return (int)e;
  }
#endif
  hipLaunchKernelGGL(kernel, grid, dim3(threads), lds, (hipStream_t)stream, p);
  OCCF_LAUNCH_CHECK();
}

static RaParams ra_params(const int64_t* g, float scale, int causal) {
  RaParams p = {};
  p.B = (int)g[0]; p.Lq = (int)g[1]; p.Lk = (int)g[2]; p.Hq = (int)g[3]; p.Hk = (int)g[4];
  p.D = (int)g[5]; p.nb = (int)g[6]; p.R = (int)g[7]; p.causal = causal != 0;
  p.qsb = g[8]; p.qsl = g[9]; p.qsh = g[10];
  p.ksb = g[11]; p.ksl = g[12]; p.ksh = g[13];
  p.vsb = g[14]; p.vsl = g[15]; p.vsh = g[16];
  p.scale = scale;
  p.c = scale * RA_LOG2E;
  return p;
}

// head dims are padded to the next multiple of 32
#define RA_DISPATCH(dtype, D, fn, ...)                         \
  do {                                                         \
    if ((dtype) == 0) {                                        \
      if ((D) <= 32) return fn<float, 32>(__VA_ARGS__);        \
      if ((D) <= 64) return fn<float, 64>(__VA_ARGS__);        \
      if ((D) <= 96) return fn<float, 96>(__VA_ARGS__);        \
      return fn<float, 128>(__VA_ARGS__);                      \
    }                                                          \
    if ((D) <= 32) return fn<ra_bf16, 32>(__VA_ARGS__);        \
    if ((D) <= 64) return fn<ra_bf16, 64>(__VA_ARGS__);        \
    if ((D) <= 96) return fn<ra_bf16, 96>(__VA_ARGS__);        \
    return fn<ra_bf16, 128>(__VA_ARGS__);                      \
  } while (0)
