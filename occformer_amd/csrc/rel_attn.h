// Shared device pieces of the attention with a bucketed relative position bias (rel_attn.hip, rel_attn_bwd.hip).
//
// Both directions are written on 32 x 32 score tiles of v_mfma_f32_32x32x16_bf16 in the orientation that keeps the
// scores in registers: the accumulator of one product is the B operand of the next.  A lane holds ONE column of the tile
// (lane & 31) and 16 of its 32 rows, row(r) = (r & 3) + 8 (r >> 2) + 4 (lane >> 5); registers 0..7 are then a B operand of
// 16 k-values {4 lk + 0..3, 8 + 4 lk + 0..3}, registers 8..15 the next 16.  The A operand of that second product is the tile
// transposed: ds_read_b64_tr_b16 hands the lanes of a 16-lane group one column each of a 4 x 16 block of the row image, in just
// this order, so that a tile lies in LDS once, as rows.
//
// Products: bf16 inputs are one product.  fp32 inputs are split into three bf16 pieces (x = h + m + l, 24 bits) and a
// product is the six terms above 2^-24; the two-piece, three-term form the other attention kernels use leaves 3e-6 ... 5e-6
// of error, which the position bias' gradient (sums with cancellation) would show.
//
// An infinity has no second and third piece (inf - inf), and as a first piece it meets the other operand's second, which may be zero
// or of the other sign.  What is loaded from q, k, v and dO is therefore split with its first two pieces kept finite: what is left
// over, infinite or NaN, is the third piece, which meets the other operand's first piece alone.  So are values that round to a bf16
// infinity (beyond 3.39e38, the lowest fp32 number as a mask among them).  Finite values up to there keep their bits.  Left: a
// product that passes the largest float 2^9 times over may be NaN instead of an infinity.
#pragma once
#include "occf_common.h"

#define RA_LOG2E 1.44269504088896340736f
#define RA_PAD 64               // bias columns kept beyond either end of the clamped distances

#ifdef OCCF_EMU
#define ra_mfma16(a, b, c) emu_mfma_f32_16x16x32_bf16(a, b, c)
#define RA_WAVE_SYNC() hipemu::wave_sync()
#define RA_WAIT_LOADS() do { } while (0)
#define RA_PRIO(n) do { } while (0)
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
// every load so far has arrived.  Operands that a loop keeps are loaded, then waited for, in front of it: left to the first use
// inside, the wait is repeated in every round and takes the next tile's loads with it.  No branch stands between such loads and
// the loop (tiles behind the last are loaded as no rows), or the wait is found missing on a path that is never taken
#define RA_WAIT_LOADS() __builtin_amdgcn_s_waitcnt(0x0F70)             // vmcnt(0)
// the wave that has products to issue goes first, so that the matrix pipe works while another wave of the SIMD does its scores
#define RA_PRIO(n) __builtin_amdgcn_s_setprio(n)
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

// bf16 rows times values in two pieces
__device__ __forceinline__ f32x16 ra_mm(const RaFrag<1>& a, const RaFrag<2>& b, f32x16 c) {
  c = occf_mfma_bf16_32x32x16(a.p[0], b.p[1], c);
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
  if constexpr (NT >= 2) {
    a -= occf_u2f(w[0] << 16);
    b -= occf_u2f(w[0] & 0xFFFF0000u);
    w[1] = occf_bf16_pack2(a, b);
  }
  if constexpr (NT == 3) {
    a -= occf_u2f(w[1] << 16);
    b -= occf_u2f(w[1] & 0xFFFF0000u);
    w[2] = occf_bf16_pack2(a, b);
  }
}

// the same of values from memory, which may be infinite: the first two pieces finite
__device__ __forceinline__ float ra_clamp(float x, float most) {
#ifdef OCCF_EMU
  return x != x ? -most : fminf(fmaxf(x, -most), most);
#else
  return __builtin_amdgcn_fmed3f(x, -most, most);
#endif
}
__device__ __forceinline__ void ra_split2_any(float a, float b, uint32_t (&w)[3]) {
  const float h = 0x1.FEp127f, m = 0x1p120f;             // the largest bf16; the most that rounding a finite value to it leaves
  w[0] = occf_bf16_pack2(ra_clamp(a, h), ra_clamp(b, h));
  a -= occf_u2f(w[0] << 16);
  b -= occf_u2f(w[0] & 0xFFFF0000u);
  w[1] = occf_bf16_pack2(ra_clamp(a, m), ra_clamp(b, m));
  a -= occf_u2f(w[1] << 16);
  b -= occf_u2f(w[1] & 0xFFFF0000u);
  w[2] = occf_bf16_pack2(a, b);
}
template <bool ANY>
__device__ __forceinline__ void ra_split2_of(float a, float b, uint32_t (&w)[3]) {
  if constexpr (ANY) ra_split2_any(a, b, w);
  else ra_split2<3>(a, b, w);
}
// does a value of a wave need that: tiles on their way into LDS are looked at in half an instruction a value (v_max3 of the
// magnitudes), and split without the clamps, which cost two each, where none does (forward and backward of 2 x 1000 fp32 rows,
// 8 heads of 24: 99.7 us without infinities' meaning, 101.4 so, 104.5 with the clamps throughout)
__device__ __forceinline__ float ra_max3(float m, uint32_t a, uint32_t b) {
#ifdef OCCF_EMU
  return fmaxf(m, fmaxf(fabsf(occf_u2f(a)), fabsf(occf_u2f(b))));
#else
  asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(m) : "v"(a), "v"(b));
  return m;
#endif
}
__device__ __forceinline__ bool ra_large(float m) { return __ballot(m > 0x1.FEp127f) != 0; }

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

// eight consecutive register values -> B operand (ANY: eight from memory, fp32)
template <int NT, bool ANY = false>
__device__ __forceinline__ RaFrag<NT> ra_pack8(const float* v) {
  uint32_t w[4][NT];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (NT == 3) ra_split2_of<ANY>(v[2 * e], v[2 * e + 1], w[e]);
    else ra_split2<NT>(v[2 * e], v[2 * e + 1], w[e]);
  }
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
    return ra_pack8<3, true>(f);
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

// LDS image of a tile's rows, one per piece.  The stride is an odd number of 16-byte units, so that the 16 rows of a b128 read lie
// on different bank quads; 304 for 128 columns (not 272), so that the 8 rows x 64 bytes of a transposing read spread over all 64
// banks too.
template <int DP> struct RaRow {
  static constexpr int LD = DP == 128 ? 304 : DP * 2 + 16;
  static constexpr int bytes(int rows) { return rows * LD; }
};

typedef uint32_t ra_u2 __attribute__((ext_vector_type(2)));

// bounded loads (no branch a load: under branches every load is waited for where the paths meet).  The resource starts at the
// tile's first row, so that 32-bit offsets reach it wherever it lies; a tile's rows span less than 2 GiB (ra_check, ra_bwd_check)
#ifdef OCCF_EMU
static inline RaU4 ra_buf16(occf_bbuf b, uint32_t off) {
  const occf_u32x4 v = occf_bbuf_load_b128(b, off);
  return RaU4{{v.x, v.y, v.z, v.w}};
}
static inline float ra_buf4(occf_bbuf b, uint32_t off) {
  float v = 0.f;
  if ((uint64_t)off + 4u <= (uint64_t)b.nbytes) memcpy(&v, b.base + off, 4);
  return v;
}
#else
__device__ __forceinline__ RaU4 ra_buf16(occf_bbuf b, uint32_t off) {
  return __builtin_bit_cast(RaU4, __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, 0));
}
__device__ __forceinline__ float ra_buf4(occf_bbuf b, uint32_t off) {
  return occf_u2f(__builtin_amdgcn_raw_buffer_load_b32(b, off, 0, 0));
}
#endif
// the next `rows` rows from `tile`: the resource ends with the last of them (rows lie D or more apart, ra_check), so that the
// rows behind read as zeros without a test
template <class T>
__device__ __forceinline__ occf_bbuf ra_tile(const T* tile, long stride, int rows, int D) {
  const int n = rows < 64 ? rows : 64;
  return occf_make_bbuf(tile, n > 0 ? ((uint32_t)(n - 1) * (uint32_t)stride + (uint32_t)D) * (uint32_t)sizeof(T) : 0u);
}

// A tile of ROWS x DP in 16-byte pieces of rows, NU of them a thread of TH: byte offsets (columns at or behind D lie outside any
// tile), loads, and the way into the row image
template <class T, int DP, int ROWS, int TH>
struct RaTileRegs {
  static constexpr int C = 16 / sizeof(T), PER = DP / C, NB = ROWS * PER, NU = (NB + TH - 1) / TH, NT = RaType<T>::NT;
  // whole rows a step of the workgroup: the pieces of a thread lie a constant apart
  static constexpr bool EVEN = TH % PER == 0;
  RaU4 x[NU];
  uint32_t at[EVEN ? 1 : NU];
  __device__ __forceinline__ void place(long stride, int D, int tid) {
#pragma unroll
    for (int n = 0; n < (EVEN ? 1 : NU); ++n) {
      const int u = tid + n * TH, row = u / PER, c = (u % PER) * C;
      at[n] = c < D && u < NB ? ((uint32_t)row * (uint32_t)stride + (uint32_t)c) * (uint32_t)sizeof(T) : OCCF_BUF_OOB;
    }
  }
  __device__ __forceinline__ void load(const T* tile, long stride, int rows, int D) {
    const occf_bbuf buf = ra_tile(tile, stride, rows < ROWS ? rows : ROWS, D);
#pragma unroll
    for (int n = 0; n < NU; ++n)
      x[n] = ra_buf16(buf, EVEN ? at[0] + n * (TH / PER) * ((uint32_t)stride * (uint32_t)sizeof(T)) : at[EVEN ? 0 : n]);
  }
  __device__ __forceinline__ void store(char* img, int tid) const {
    if (NT == 3 && ra_large(largest())) put<true>(img, tid);
    else put<false>(img, tid);
  }
  __device__ __forceinline__ float largest() const {
    float m = 0.f;
#pragma unroll
    for (int n = 0; n < NU; ++n) m = ra_max3(ra_max3(m, x[n].x[0], x[n].x[1]), x[n].x[2], x[n].x[3]);
    return m;
  }
  template <bool ANY>
  __device__ __forceinline__ void put(char* img, int tid) const {
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      const int u = tid + n * TH, row = u / PER, c = (u % PER) * C;
      if (NB % TH && u >= NB) break;
      char* to = img + row * RaRow<DP>::LD + c * 2;
      if constexpr (NT == 1) {
        *(bf16x8*)to = ra_as_frag(x[n].x[0], x[n].x[1], x[n].x[2], x[n].x[3]);
      } else {
        uint32_t a[3], b[3];
        ra_split2_of<ANY>(occf_u2f(x[n].x[0]), occf_u2f(x[n].x[1]), a);
        ra_split2_of<ANY>(occf_u2f(x[n].x[2]), occf_u2f(x[n].x[3]), b);
#pragma unroll
        for (int t = 0; t < 3; ++t) {
          const ra_u2 w = {a[t], b[t]};
          *(ra_u2*)(to + t * RaRow<DP>::bytes(ROWS)) = w;
        }
      }
    }
  }
};

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
template <bool ANY>
__device__ __forceinline__ RaFrag<1> ra_raw_frag(const RaRaw<ra_bf16>& w) {
  RaFrag<1> f;
  f.p[0] = ra_as_frag(w.x[0].x[0], w.x[0].x[1], w.x[0].x[2], w.x[0].x[3]);
  return f;
}
template <bool ANY>
__device__ __forceinline__ RaFrag<3> ra_raw_frag(const RaRaw<float>& w) {
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = occf_u2f(w.x[e >> 2].x[e & 3]);
  return ra_pack8<3, ANY>(f);
}
// ds_read_b64_tr_b16: lane 4 r + q of a 16-lane group gives the address of row r, columns 4 q .. 4 q + 3 of a 4 x 16 block;
// lane t gets column t, rows 0..3
#ifdef OCCF_EMU
static inline ra_u2 ra_read_tr(const char* at) {
  struct V { uint16_t e[4]; } v;
  memcpy(&v, at, 8);
  const int lane = threadIdx.x & 63, t = lane & 15;
  uint32_t r[4];
  for (int e = 0; e < 4; ++e) r[e] = hipemu::lane_exchange(v, (lane & 48) + 4 * e + (t >> 2)).e[t & 3];
  return ra_u2{r[0] | (r[1] << 16), r[2] | (r[3] << 16)};
}
#else
typedef short ra_s4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ ra_u2 ra_read_tr(const char* at) {
  return __builtin_bit_cast(ra_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ra_s4*)at));
}
#endif

// A operand: 32 rows from row0, k step ks of 16 columns
template <int NT, int DP, int ROWS>
__device__ __forceinline__ RaFrag<NT> ra_read_row(const char* img, int row0, int ks, int li, int lk) {
  RaFrag<NT> f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
    f.p[t] = *(const bf16x8*)(img + t * RaRow<DP>::bytes(ROWS) + (row0 + li) * RaRow<DP>::LD + ks * 32 + lk * 16);
  return f;
}
// A operand, transposed: 32 columns of the tile from c0, k step ks of 16 tile rows
template <int NT, int DP, int ROWS>
__device__ __forceinline__ RaFrag<NT> ra_read_trans(const char* img, int c0, int ks, int lane) {
  RaFrag<NT> f;
  const int row = 4 * (lane >> 5) + ((lane & 15) >> 2), col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  const char* at = img + row * RaRow<DP>::LD + col * 2 + ks * 16 * RaRow<DP>::LD + c0 * 2;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const ra_u2 a = ra_read_tr(at + t * RaRow<DP>::bytes(ROWS)), b = ra_read_tr(at + t * RaRow<DP>::bytes(ROWS) + 8 * RaRow<DP>::LD);
    f.p[t] = ra_as_frag(a.x, a.y, b.x, b.y);
  }
  return f;
}
// the same for the 16-column form: 16 columns of the tile from c0, its 32 rows
template <int NT, int DP>
__device__ __forceinline__ RaFrag<NT> ra_read_trans16(const char* img, int c0, int lane) {
  RaFrag<NT> f;
  const char* at = img + (4 * (lane >> 4) + ((lane & 15) >> 2)) * RaRow<DP>::LD + (c0 + 4 * (lane & 3)) * 2;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const ra_u2 a = ra_read_tr(at + t * RaRow<DP>::bytes(32)), b = ra_read_tr(at + t * RaRow<DP>::bytes(32) + 16 * RaRow<DP>::LD);
    f.p[t] = ra_as_frag(a.x, a.y, b.x, b.y);
  }
  return f;
}

// ---- the same chain on 16 columns (v_mfma_f32_16x16x32_bf16): a lane holds column lane & 15 and, of 32 tile rows in two
// accumulators, rows 16 (e >> 2) + 4 (lane >> 4) + (e & 3), e = 0..7, which are one B operand of 32 k-values.
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

// bf16 rows times values in two pieces
__device__ __forceinline__ f32x4 ra_mm16(const RaFrag<1>& a, const RaFrag<2>& b, f32x4 c) {
  c = ra_mfma16(a.p[0], b.p[1], c);
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

// biases of head h behind either end of the distances
template <class T>
__device__ __forceinline__ void ra_far_bias(const RaParams& p, int h, float& below, float& above) {
  const T* table = (const T*)p.table;
  below = ra_bias(ra_to_float(table[(long)occf_clampi(p.lut[0], p.nb - 1) * p.Hq + h]));
  above = ra_bias(ra_to_float(table[(long)occf_clampi(p.lut[2 * p.R], p.nb - 1) * p.Hq + h]));
#ifndef OCCF_EMU
  below = occf_u2f(occf_wave_uniform(occf_f2u(below)));
  above = occf_u2f(occf_wave_uniform(occf_f2u(above)));
#endif
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
  nq = occf_wave_uniform(nq);                            // scalar loop bounds and branches
  nk = occf_wave_uniform(nk);
  start = occf_wave_uniform(start);
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
  if (Hq * Lq >= (1L << 29) || Lq * (Hq / Hk) >= (1L << 30) || B * Hk * ((Lq * (Hq / Hk) + 31) / 32) * 64 >= 2147483647L) return OCCF_ESHAPE;
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
