// Attention with a learned relative position bias by buckets: forward.
//
//   t_ij = scale q_i.k_j + T[bucket(j - p_i), h],  p_i = q_start + i;   o_i = sum_j softmax_j(t_ij) v_j
//
// over the pairs that count (j < k_len, i < q_len, and j <= p_i when causal).  The reference has a learned position bias in
// its window attention only (projects/mmdet3d_plugin/occformer/backbones/modules/window_attention.py:69-107: a table over the
// 169 offsets of a 7 x 7 window); here the distance is any length and the table has one row a bucket of distances.
//
// Neither the scores nor the bias exist in memory.  The bucket function is a table over the clamped distance (-R .. R), so a
// head's bias is 2 R + 1 floats in LDS: a 32 x 32 score tile wholly further than R from the diagonal adds a constant (folded
// into the exponent's fma), any other reads its 16 values a lane at constant offsets from one address.
#include "rel_attn.h"
#include "../../include/occformer_hip.h"

#define RA_EXCEED 8.0f          // the running maximum follows only when a tile exceeds it by 2^8: p <= 256, sums stay fp32

// ---------------------------------------------------------------------------------------------------------------------
// Many queries: a workgroup owns 128 queries of one head, a wave 32 of them (a lane one query: its running maximum and sum
// are registers), and walks the keys in tiles of KT through LDS; the next tile's rows travel from memory meanwhile.  Two
// workgroups a compute unit: one's exponentials run beside the other's products.  2 x 4096 causal rows, 16 heads of 64: 95 us,
// 720 TFLOP/s of the two products; 8192 rows, 16 heads of 128: 308 us, 890 TFLOP/s.  Of that time the matrix pipes are busy 30 and
// 39 %, vector instructions 52 and 35, the LDS 32 and 40: bound by a wave's chain from scores over exponentials to the second product,
// which two waves a SIMD fill in part.  Tried at these two (at 104 and 330 us; comparisons are of short runs, in which the card has
// not reached its clock): a second image and one barrier a tile, 115 and 436 (the offsets cost a
// wave a SIMD); tiles of 32 keys, 165 and 434; probabilities in two bf16 pieces, 134 and 427 against 312, so that bf16 ones go into
// their product (not into their sum) rounded to bf16: the output is off by 2.1e-3 where its own rounding is 1.7e-3; Q K^T of the next tile in one block with this one's exponentials, 144 and 567.
template <class T, int DP, int KT>
struct RaFwd {
  static constexpr int tile = 2 * RaType<T>::NT * RaRow<DP>::bytes(KT);                  // K and V
  static size_t bytes(int R) { return tile + 4 * (2 * (size_t)R + 1 + 2 * RA_PAD); }
};

template <class T, int DP, int KT>
__global__ void __launch_bounds__(256, RaType<T>::NT == 1 || DP <= 64 ? 2 : 1) rel_attn_fwd_kernel(RaParams p) {
  constexpr int NT = RaType<T>::NT, KS = DP / 16, DT = DP / 32;
  OCCF_DYN_SMEM(smem);
  float* lut = (float*)(smem + RaFwd<T, DP, KT>::tile);

  const int tid = threadIdx.x, wave = occf_wave_uniform(tid >> 6), lane = tid & 63, li = lane & 31, lk = lane >> 5;
  const int nqt = (p.Lq + 127) / 128;
  int qt, bh;
  ra_order(p, blockIdx.x, nqt, p.B * p.Hq, qt, bh);
  qt = nqt - 1 - qt;                                     // the last queries see the most keys
  const int h = bh % p.Hq, b = bh / p.Hq;
  const int hk = h / (p.Hq / p.Hk);
  int nq, nk, start;
  ra_lengths(p, b, nq, nk, start);

  ra_fill_bias<T>(lut, p, h, tid, 256);
  float far_below, far_above;
  ra_far_bias<T>(p, h, far_below, far_above);

  const T* kb = (const T*)p.k + (long)b * p.ksb + (long)hk * p.ksh;
  const T* vb = (const T*)p.v + (long)b * p.vsb + (long)hk * p.vsh;

  RaTileRegs<T, DP, KT, 256> rk, rv;
  rk.place(p.ksl, p.D, tid);
  rv.place(p.vsl, p.D, tid);

  const int i0 = qt * 128 + wave * 32, i = i0 + li;
  const int pi = start + i;
  const T* qrow = (const T*)p.q + (long)b * p.qsb + (long)occf_clampi(i, p.Lq - 1) * p.qsl + (long)h * p.qsh;
  RaFrag<NT> qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int d = ks * 16 + lk * 8;
    qf[ks] = ra_row_frag<T>(qrow + (d < p.D ? d : 0), i < nq && d < p.D);
  }

  // keys of this workgroup: all, or up to its last query's position
  int kend = nk;
  if (p.causal) {
    const int last = start + (qt * 128 + 128 < nq ? qt * 128 + 128 : nq);      // behind the last query
    kend = last < kend ? (last > 0 ? last : 0) : kend;
  }
  if (qt * 128 >= nq) kend = 0;
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = ra_zero16();
  float m = -INFINITY, mref = 0.f, l = 0.f;

  const auto load = [&](int k0) {
    rk.load(kb + k0 * p.ksl, p.ksl, kend - k0, p.D);
    rv.load(vb + k0 * p.vsl, p.vsl, kend - k0, p.D);
  };
  const char *img_k = smem, *img_v = smem + NT * RaRow<DP>::bytes(KT);
  const int ntile = (kend + KT - 1) / KT;
  load(0);
  RA_WAIT_LOADS();
  for (int kt = 0; kt < ntile; ++kt) {
    const int k0 = kt * KT;
    __syncthreads();                                     // no wave reads the last tile any more
    rk.store(smem, tid);
    rv.store(smem + NT * RaRow<DP>::bytes(KT), tid);
    __syncthreads();
    load(k0 + KT);
    if (i0 >= nq || (p.causal && k0 > start + i0 + 31)) continue;      // wave-uniform
    f32x16 s[KT / 32];
    RA_PRIO(1);
#pragma unroll
    for (int sub = 0; sub < KT / 32; ++sub) {
      s[sub] = ra_zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        s[sub] = ra_mm<NT>(ra_read_row<NT, DP, KT>(img_k, sub * 32, ks, li, lk), qf[ks], s[sub]);
    }
    RA_PRIO(0);
    float mx = -INFINITY, ce[KT / 32], be[KT / 32];
#pragma unroll
    for (int sub = 0; sub < KT / 32; ++sub) {
      const int j0 = k0 + sub * 32, rel0 = j0 - (start + i0);           // tile distances: rel0 - 31 .. rel0 + 31
      const int jl = j0 + 4 * lk;
      const bool near = rel0 - 31 < p.R && rel0 + 31 > -p.R;
      ra_bias_mask<1>(s[sub], lut + (near ? jl - pi + p.R + RA_PAD : 0), near, rel0 > 0 ? far_above : far_below,
                      j0 + 32 > kend || (p.causal && rel0 + 31 > 0), p.c, ce[sub], be[sub],
                      [&](int o) { return jl + o >= kend || (p.causal && jl + o > pi); });
      float x = s[sub][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) x = fmaxf(x, s[sub][r]);
      mx = fmaxf(mx, fmaf(x, ce[sub], be[sub]));
    }
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    if (__ballot(mx > m + RA_EXCEED)) {
      const float mn = fmaxf(m, mx);
      const float a = ra_exp2(m - (mn == -INFINITY ? 0.f : mn));       // first keys of a row: exp2(-inf) = 0
      m = mn;
      mref = mn == -INFINITY ? 0.f : mn;
      l *= a;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[dt][r] *= a;
    }
    // a tile's probabilities first: added one by one onto the row's sum each would round at its size (relative error over 32768
    // keys, restated in numpy: 1.2e-6 one by one, 2e-7 by tiles)
    float sum = 0.f;
#pragma unroll
    for (int sub = 0; sub < KT / 32; ++sub) {
      float pv[16];
      const float off = be[sub] - mref;
#pragma unroll
      for (int r = 0; r < 16; ++r) pv[r] = ra_exp2(fmaf(s[sub][r], ce[sub], off));
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += pv[r];
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const RaFrag<NT> pf = ra_pack8<NT>(pv + s2 * 8);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          acc[dt] = ra_mm<NT>(ra_read_trans<NT, DP, KT>(img_v, dt * 32, sub * 2 + s2, lane), pf, acc[dt]);
      }
    }
    l += sum;
  }
  l += __shfl_xor(l, 32);
  if (i >= p.Lq) return;
  const bool some = l != 0.f && i < nq;                   // rows behind the last query went along with their tile
  const float inv = some ? 1.0f / l : 0.f;
  if (!some) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = ra_zero16();
  }
  T* orow = (T*)p.o + (((long)b * p.Lq + i) * p.Hq + h) * p.D;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = dt * 32 + 8 * g + 4 * lk;
      if (d < p.D)
        ra_store4(orow + d, acc[dt][4 * g] * inv, acc[dt][4 * g + 1] * inv, acc[dt][4 * g + 2] * inv, acc[dt][4 * g + 3] * inv);
    }
  if (p.lse && lk == 0) p.lse[((long)b * p.Hq + h) * p.Lq + i] = some ? m + ra_log2(l) : -INFINITY;
}

// ---------------------------------------------------------------------------------------------------------------------
// Parts by the sequences' own lengths.  Equal parts of the longest leave the card half empty when lengths differ (16 sequences
// of 0 ... 8192 keys: 72 us at 4 parts each), and many small ones cost about 10 us a workgroup to begin and end.  So the keys of
// all sequences are counted, a part is their share of nsplit B parts (in steps of 128), and sequence b gets ceil(len_b / part)
// consecutive units of the B nsplit + B there are at most.  `unit` >= 0: which sequence and part it is (false: none);
// else `seq`: its first unit (in `split`) and their number n.  One wave's lanes hold 64 sequences at a time.
__device__ __forceinline__ bool ra_unit(const RaParams& p, int unit, int seq, int& b, int& split, int& n, int& chunk) {
  const int lane = threadIdx.x & 63;
  long total = 0;
  for (int s0 = 0; s0 < p.B; s0 += 64) {
    int x = s0 + lane < p.B ? occf_clampi(p.k_lens[s0 + lane], p.Lk) : 0;
    long y = x;
#pragma unroll
    for (int mm = 32; mm > 0; mm >>= 1) y += __shfl_xor(y, mm);
    total += y;
  }
  const long parts = (long)p.B * p.nsplit;
  chunk = (int)(((total + parts - 1) / parts + 127) / 128 * 128);
  chunk = chunk < 128 ? 128 : chunk;
  int before = 0;
  for (int s0 = 0; s0 < p.B; s0 += 64) {
    const int x = s0 + lane < p.B ? occf_clampi(p.k_lens[s0 + lane], p.Lk) : 0;
    const int c = (x + chunk - 1) / chunk;
    int sum = c;                                         // units up to and with this lane's sequence
#pragma unroll
    for (int mm = 1; mm < 64; mm <<= 1) {
      const int y = __shfl_up(sum, mm);
      if (lane >= mm) sum += y;
    }
    sum += before;
    if (unit >= 0) {
      const int at = __popcll(__ballot(sum <= unit));
      if (at < 64 && s0 + at < p.B) {
        b = s0 + at;
        n = __shfl(c, at);
        split = unit - (__shfl(sum, at) - n);
        return true;
      }
    } else if (seq < s0 + 64) {
      n = __shfl(c, seq - s0);
      split = __shfl(sum, seq - s0) - n;
      return true;
    }
    before = __shfl(sum, 63);
  }
  return false;
}

// Few queries: the rows of one key head (query i of its G query heads, row = i G + g) in groups of RW = 32, or 16 where there are
// no more, share every key that is read.  The keys are split over workgroups and, tile by tile, over a workgroup's four waves;
// a wave reads its key rows straight into operand registers and takes its value rows through LDS of its own, so that no wave
// waits for another before the join at the end.  (Keys through LDS, in whole rows of the cache line, took 99 instead of 67 us for
// 4 x 2500 fp32 queries and as long for single ones.)  Bound by the stream of keys and values: 16 rows take half the
// accumulators, products and exponentials of 32, which leaves room for a second tile in flight.  16 sequences of up to 8192 bf16
// keys, 8 key heads of 128: 59 us, 4.8 TB/s, and 8.5 for the join; 4 x 2500 fp32 queries and keys, 4 heads of 32: 58 us, vector
// instructions busy 55 % of it (a score's bias, exponential and pieces, the keys' splitting), the matrix pipes 23 %.
// bf16: probabilities go into their product as two bf16 pieces (2^-16), which the stream hides: 67.2 us for the single queries
// above either way, 86.4 instead of 85.9 for forward and backward of 3 x 777 rows, 12 heads of 64.
// part != NULL: unnormalised sums, maxima and sums of exponentials of a split.
template <class T, int DP, int RW>
struct RaFew {
  static constexpr int NT = RaType<T>::NT, NW = 4, VT = NT * RaRow<DP>::bytes(32);
  static constexpr int join = RW * (DP + 4) * 4;         // [RW rows][DP + 4] floats of one wave
  static constexpr int wave = VT > join ? VT : join;
  static size_t bytes(int nb, int R) { return NW * wave + 4 * ((size_t)nb * RW + 2 * R + 1 + (2 * NW + 2) * RW); }
};

template <class T, int DP, int RW>
__global__ void __launch_bounds__((RaFew<T, DP, RW>::NW * 64), RaType<T>::NT == 1 || DP <= 32 ? 2 : 1)
    rel_attn_few_kernel(RaParams p) {
  constexpr int NT = RaType<T>::NT, NW = RaFew<T, DP, RW>::NW, TH = NW * 64;
  constexpr int NE = RW / 2;                             // scores of a 32-key tile a lane holds
  constexpr int QS = DP / (RW == 32 ? 16 : 32);          // k steps of Q K^T
  constexpr int KR = DP / 16;                            // key fragments: [k step] or [16-key half][k step]
  constexpr int DT = DP / RW;                            // column tiles of the output
  typedef typename std::conditional<RW == 32, f32x16, f32x4>::type Acc;
  OCCF_DYN_SMEM(smem);
  const int tid = threadIdx.x, wave = occf_wave_uniform(tid >> 6), lane = tid & 63, li = lane & (RW - 1), lg = lane / RW;
  char* img_v = smem + wave * RaFew<T, DP, RW>::wave;
  float* tab = (float*)(smem + NW * RaFew<T, DP, RW>::wave);            // [nb][RW] bias of row li
  int* lut = (int*)(tab + p.nb * RW);                                   // [2 R + 1] bucket of a distance
  float* stat = (float*)(lut + 2 * p.R + 1);                            // [2 NW + 2][RW]
  const auto key_of = [&](int e) { return RW == 32 ? (e & 3) + 8 * (e >> 2) + 4 * lg : 16 * (e >> 2) + 4 * lg + (e & 3); };

  const int G = p.Hq / p.Hk, rows = p.Lq * G, nrt = (rows + RW - 1) / RW;
  int rt, bh, b, split, chunk = p.chunk;
  ra_order(p, blockIdx.x, nrt, p.units * p.Hk, rt, bh);
  rt = nrt - 1 - rt;                                     // the last queries see the most keys
  // split walks: units go round the XCDs and every XCD sees all heads (rows of one head are a fixed 256 bytes of a wider row, and
  // an L2's 16 channels are 256 bytes wide: one head alone would keep two of them busy)
  int hk, unit;
  if (p.part) {
    hk = bh / p.units;
    unit = bh - hk * p.units;
  } else {
    unit = bh / p.Hk;
    hk = bh - unit * p.Hk;
  }
  if (p.by_length) {
    int n;
    if (!ra_unit(p, unit, -1, b, split, n, chunk)) return;
    b = occf_wave_uniform(b);                            // (came by shuffles: addresses of scalar resources)
    split = occf_wave_uniform(split);
    chunk = occf_wave_uniform(chunk);
  } else {
    b = unit / p.nsplit;
    split = unit - b * p.nsplit;
  }
  int nq, nk, start;
  ra_lengths(p, b, nq, nk, start);
  const int row = rt * RW + li;
  const int i = row / G, h = hk * G + row % G;
  const bool live = row < rows && i < nq;
  const int pi = start + i;
  const int i_first = (rt * RW) / G, i_last = (rt * RW + RW - 1 < rows ? rt * RW + RW - 1 : rows - 1) / G;
  int kend = nk;
  if (p.causal) {
    const int last = start + (i_last < nq ? i_last : nq - 1) + 1;
    kend = last < kend ? (last > 0 ? last : 0) : kend;
  }
  if (i_first >= nq) kend = 0;
  const int first = split * chunk;
  const int lim = first + chunk < kend ? first + chunk : kend;
  const T* kb = (const T*)p.k + (long)b * p.ksb + (long)hk * p.ksh;
  const T* vb = (const T*)p.v + (long)b * p.vsb + (long)hk * p.vsh;

  // the first tile is on its way before the tables are made
  RaRaw<T> rk[KR];
  RaTileRegs<T, DP, 32, 64> rv;
  rv.place(p.vsl, p.D, lane);
  const int jw = first + wave * 32;                      // the wave's first tile
  uint32_t at_k[KR];
#pragma unroll
  for (int n = 0; n < KR; ++n)
    at_k[n] = RW == 32 ? ra_raw_at<T>(p.ksl, p.D, li, n * 16 + lg * 8)
                       : ra_raw_at<T>(p.ksl, p.D, (n / QS) * 16 + li, (n % QS) * 32 + lg * 8);
  auto load = [&](int j) {
    const occf_bbuf tk = ra_tile(kb + j * p.ksl, p.ksl, lim - j < 32 ? lim - j : 32, p.D);
#pragma unroll
    for (int n = 0; n < KR; ++n) ra_load_raw<T>(rk[n], tk, at_k[n]);
    rv.load(vb + j * p.vsl, p.vsl, lim - j, p.D);
  };
  load(jw);

  const T* qrow = (const T*)p.q + (long)b * p.qsb + (long)(live ? i : 0) * p.qsl + (long)(live ? h : 0) * p.qsh;
  RaFrag<NT> qf[QS];
#pragma unroll
  for (int ks = 0; ks < QS; ++ks) {
    const int d = (ks * (64 / RW) + lg) * 8;
    qf[ks] = ra_row_frag<T>(qrow + (d < p.D ? d : 0), live && d < p.D);
  }
  RA_WAIT_LOADS();
  if (first < lim) {
    for (int t = tid; t < p.nb * RW; t += TH) {
      const int r = rt * RW + t % RW;
      tab[t] = r < rows ? ra_bias(ra_to_float(((const T*)p.table)[(long)(t / RW) * p.Hq + hk * G + r % G])) : 0.f;
    }
    for (int t = tid; t < 2 * p.R + 1; t += TH) lut[t] = occf_clampi(p.lut[t], p.nb - 1) * RW;
  }
  __syncthreads();

  Acc acc[DT];
  float m, mref, l;
  const auto walk = [&](auto any) {
    constexpr bool ANY = decltype(any)::value;           // with infinities (ra_split2_any)
    constexpr int NP = NT == 3 ? 3 : ANY ? 1 : 2;        // pieces of a probability
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < RW * RW / 64; ++r) acc[dt][r] = 0.f;
    m = -INFINITY;
    mref = l = 0.f;
    for (int j0 = jw; j0 < lim; j0 += NW * 32) {
      float s[NE];
      RA_WAVE_SYNC();
      rv.template put<ANY>(img_v, lane);
      RA_WAVE_SYNC();
      if constexpr (RW == 32) {
        f32x16 x = ra_zero16();
#pragma unroll
        for (int ks = 0; ks < QS; ++ks) x = ra_mm<NT>(ra_raw_frag<ANY>(rk[ks]), qf[ks], x);
#pragma unroll
        for (int e = 0; e < NE; ++e) s[e] = x[e];
      } else {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < QS; ++ks) x = ra_mm16<NT>(ra_raw_frag<ANY>(rk[hf * QS + ks]), qf[ks], x);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[hf * 4 + e] = x[e];
        }
      }
      load(j0 + NW * 32);

      const int lo = j0 - (start + i_last), hi = j0 + 31 - (start + i_first);        // distances of the tile
      float mx = -INFINITY;
      if (hi <= -p.R || lo >= p.R) {
        const float far = tab[lut[hi <= -p.R ? 0 : 2 * p.R] + li];
#pragma unroll
        for (int e = 0; e < NE; ++e) s[e] = fmaf(s[e], p.c, far);
      } else {
#pragma unroll
        for (int e = 0; e < NE; ++e)
          s[e] = fmaf(s[e], p.c, tab[lut[occf_clampi(j0 + key_of(e) - pi + p.R, 2 * p.R)] + li]);
      }
      if (j0 + 32 > lim || (p.causal && j0 + 31 > start + i_first)) {
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          const int j = j0 + key_of(e);
          s[e] = j >= lim || (p.causal && j > pi) ? -INFINITY : s[e];
        }
      }
#pragma unroll
      for (int e = 0; e < NE; ++e) mx = fmaxf(mx, s[e]);
#pragma unroll
      for (int mm = RW; mm < 64; mm <<= 1) mx = fmaxf(mx, __shfl_xor(mx, mm));
      if (__ballot(mx > m + RA_EXCEED)) {
        const float mn = fmaxf(m, mx);
        const float a = ra_exp2(m - (mn == -INFINITY ? 0.f : mn));
        m = mn;
        mref = mn == -INFINITY ? 0.f : mn;
        l *= a;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < RW * RW / 64; ++r) acc[dt][r] *= a;
      }
      float pv[NE];
#pragma unroll
      for (int e = 0; e < NE; ++e) pv[e] = ra_exp2(s[e] - mref);
      float sum = 0.f;                                   // (as in the kernel for many queries)
#pragma unroll
      for (int e = 0; e < NE; ++e) sum += pv[e];
      l += sum;
#pragma unroll
      for (int s2 = 0; s2 < NE / 8; ++s2) {
        const RaFrag<NP> pf = ra_pack8<NP>(pv + s2 * 8);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          if constexpr (RW == 32) acc[dt] = ra_mm(ra_read_trans<NT, DP, 32>(img_v, dt * 32, s2, lane), pf, acc[dt]);
          else acc[dt] = ra_mm16(ra_read_trans16<NT, DP>(img_v, dt * 16, lane), pf, acc[dt]);
        }
      }
    }
  };
  walk(std::false_type());
  // an infinite (fp32: or nearly infinite) key or value leaves NaN behind: inf - inf among its pieces, or inf times a second piece of
  // zero.  This wave's keys once more, then, split for them, bf16 probabilities in one piece (looking for them ahead of each tile
  // costs 4.5 % at 4 x 2500 fp32 queries and keys, 4 heads of 32; so it is 1.8 %)
  bool bad = l != l;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < RW * RW / 64; ++r) bad |= acc[dt][r] != acc[dt][r];
  if (__ballot(bad)) {
    load(jw);
    walk(std::true_type());
  }
#pragma unroll
  for (int mm = RW; mm < 64; mm <<= 1) l += __shfl_xor(l, mm);
  if (!live || l == 0.f) {                               // rows behind the last query, or without a key here, went along with
    l = 0.f;                                             // their tile: 0 times an infinite value is no zero
    m = -INFINITY;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < RW * RW / 64; ++r) acc[dt][r] = 0.f;
  }

  // ---- join the waves: maxima and sums first, then the rescaled accumulators in wave order
  if (lg == 0) {
    stat[wave * RW + li] = m;
    stat[(NW + wave) * RW + li] = l;
  }
  __syncthreads();
  float mj = -INFINITY, lj = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) mj = fmaxf(mj, stat[w * RW + li]);
  const float mz = mj == -INFINITY ? 0.f : mj;
#pragma unroll
  for (int w = 0; w < NW; ++w) lj += stat[(NW + w) * RW + li] * ra_exp2(stat[w * RW + li] - mz);
  const float a = ra_exp2(m - mz);
  float* jo = (float*)img_v;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < RW * RW / 256; ++g)
      ra_store4(jo + li * (DP + 4) + dt * RW + 8 * g + 4 * lg, acc[dt][4 * g] * a, acc[dt][4 * g + 1] * a,
                acc[dt][4 * g + 2] * a, acc[dt][4 * g + 3] * a);
  float* joined = stat + 2 * NW * RW;
  if (wave == 0 && lg == 0) {
    joined[li] = mj;
    joined[RW + li] = lj;
  }
  __syncthreads();
  for (int u = tid; u < RW * (DP / 4); u += TH) {
    const int r = u / (DP / 4), d = (u % (DP / 4)) * 4;
    const int rw = rt * RW + r;
    if (rw >= rows || d >= p.D) continue;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float4 y = *(const float4*)((float*)(smem + w * RaFew<T, DP, RW>::wave) + r * (DP + 4) + d);
      x[0] += y.x; x[1] += y.y; x[2] += y.z; x[3] += y.w;
    }
    const float lr = joined[RW + r], mr = joined[r];
    const int ri = rw / G, rh = hk * G + rw % G;
    if (p.part) {
      float* ph = p.part + (((long)unit * p.Hk + hk) * nrt + rt) * (32 * (p.D + 2));
      ra_store4(ph + 64 + r * p.D + d, x[0], x[1], x[2], x[3]);
      if (d == 0) {
        ph[r] = mr;
        ph[32 + r] = lr;
      }
    } else {
      const float inv = lr != 0.f ? 1.0f / lr : 0.f;
      ra_store4((T*)p.o + (((long)b * p.Lq + ri) * p.Hq + rh) * p.D + d, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
      if (p.lse && d == 0) p.lse[((long)b * p.Hq + rh) * p.Lq + ri] = lr != 0.f ? mr + ra_log2(lr) : -INFINITY;
    }
  }
}

// joins the parts of rel_attn_few_kernel in their order: one thread four columns of a row, a wave of one sequence.
// All latency (the lengths, then the parts): one pass with a running maximum instead of one for the maxima and one for the sums
// (7.3 instead of 8.5 us for four parts of 512 rows of 128).
template <class T>
__global__ void __launch_bounds__(256) rel_attn_join_kernel(RaParams p) {
  const int G = p.Hq / p.Hk, rows = p.Lq * G, nrt = (rows + 31) / 32;
  const int per = rows * (p.D / 4), blocks = (per + 255) / 256;           // four columns a thread; blocks of one key head
  const int bh = blockIdx.x / blocks, u = (blockIdx.x - bh * blocks) * 256 + threadIdx.x;
  const int hk = bh % p.Hk, b = bh / p.Hk;
  int first = b * p.nsplit, n = p.nsplit;
  if (p.by_length) {
    int at = b, split, chunk;
    ra_unit(p, -1, b, at, split, n, chunk);
    first = split;
  }
  if (u >= per) return;
  const int d = u % (p.D / 4) * 4, rw = u / (p.D / 4), r = rw & 31;
  const long step = (long)p.Hk * nrt * (32 * (p.D + 2));
  const float* ph = p.part + (((long)first * p.Hk + hk) * nrt + (rw >> 5)) * (32 * (p.D + 2));
  float m = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < n; s0 += 8) {                    // eight parts' loads in flight at once
    float pm[8], pl[8];
    float4 y[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const bool ok = s0 + s < n;
      const float* at = ph + (ok ? s0 + s : n - 1) * step;
      const float4 z = *(const float4*)(at + 64 + r * p.D + d);
      pm[s] = ok ? at[r] : -INFINITY;
      pl[s] = ok ? at[32 + r] : 0.f;
      y[s] = make_float4(ok ? z.x : 0.f, ok ? z.y : 0.f, ok ? z.z : 0.f, ok ? z.w : 0.f);
    }
    float top = m;
#pragma unroll
    for (int s = 0; s < 8; ++s) top = fmaxf(top, pm[s]);
    const float mz = top == -INFINITY ? 0.f : top, old = ra_exp2(m - mz);
    m = top;
    l *= old;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= old;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const float a = ra_exp2(pm[s] - mz);
      l = fmaf(pl[s], a, l);
      x[0] = fmaf(y[s].x, a, x[0]);
      x[1] = fmaf(y[s].y, a, x[1]);
      x[2] = fmaf(y[s].z, a, x[2]);
      x[3] = fmaf(y[s].w, a, x[3]);
    }
  }
  const float inv = l != 0.f ? 1.0f / l : 0.f;
  const int i = rw / G, h = hk * G + rw % G;
  ra_store4((T*)p.o + (((long)b * p.Lq + i) * p.Hq + h) * p.D + d, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
  if (p.lse && d == 0) p.lse[((long)b * p.Hq + h) * p.Lq + i] = l != 0.f ? m + ra_log2(l) : -INFINITY;
}

// ---------------------------------------------------------------------------------------------------------------------
// How a call is run.  `walks`: workgroups of the kernel for many queries, counted by the keys they can see (causal: about half; own
// key lengths: as if half).  The few-query kernel takes those calls where there are too few to fill the card, as it cuts the work
// finer, but it reads the keys once for 32 rows instead of 128 and gains less the wider a head is.  us, few / many queries:
//   heads of 32:  288 walks, bf16  18 / 20, fp32  40 /  42;  384 walks   37 /  24,  79 /  57
//   heads of 64:  136 walks, bf16  32 / 41, fp32  74 / 105;  168 walks   23 /  18,  43 /  42
//   heads of 128:  48 walks, bf16  29 / 41, fp32  86 / 137;  64 walks    21 /  18,  50 /  45
// Its keys are cut into parts until three workgroups a compute unit are there (fp32: two, heads beyond 64 columns one, what its
// registers hold), never a round more: us, so / otherwise:  16 sequences of 8192 bf16 keys, 8 key heads of 128: 106 / 117 with two;
// 4 of 8192 fp32 keys, 4 key heads of 128: 45 / 56 with two;  2 x 400 bf16, 16 heads of 64: 12 / 23 with a part that fills half
// a round.  No part is shorter than what the launch that joins them costs: one query of 8 heads, 333 fp32 keys of 24 in one part
// 11.7, in three 15.3; 700 bf16 keys of 64 10.9 and 16; 512 fp32 keys of 128 in four 16.7, in one 25.
static void ra_plan(const int64_t* g, int causal, int lengths, int dtype, int& few, int& nsplit, int& chunk) {
  const long B = g[0], Lq = g[1], Lk = g[2], Hq = g[3], Hk = g[4], D = g[5];
  const long rows = Lq * (Hq / Hk), groups = B * Hk * ((rows + 31) / 32), nqt = (Lq + 127) / 128;
  const long walks = B * Hq * (causal ? nqt + 1 : 2 * nqt) / (lengths && B > 1 ? 4 : 2);
  few = rows <= 32 || walks < (D <= 32 ? 340 : D <= 64 ? 160 : 56);
  const long most = Lk / (dtype == 1 ? 768 : D <= 64 ? 256 : 128), want = (dtype == 1 ? 768 : D <= 64 ? 512 : 256) / groups;
  nsplit = (int)(want < most ? want : most);
  nsplit = nsplit < 1 ? 1 : (nsplit > 64 ? 64 : nsplit);
  chunk = (int)(((Lk + nsplit - 1) / nsplit + 127) / 128 * 128);
  nsplit = (int)((Lk + chunk - 1) / chunk);
}

template <class T, int DP>
static int ra_fwd(RaParams& p, int few, void* stream) {
  if (few) {
    const long rows = (long)p.Lq * (p.Hq / p.Hk), nrt = (rows + 31) / 32;
    const dim3 grid((unsigned)(p.units * p.Hk * nrt));
    const int rc = rows <= 16 ? ra_launch(rel_attn_few_kernel<T, DP, 16>, grid, RaFew<T, DP, 16>::NW * 64,
                                          RaFew<T, DP, 16>::bytes(p.nb, p.R), stream, p)
                              : ra_launch(rel_attn_few_kernel<T, DP, 32>, grid, RaFew<T, DP, 32>::NW * 64,
                                          RaFew<T, DP, 32>::bytes(p.nb, p.R), stream, p);
    if (rc || !p.part) return rc;
    const long blocks = (rows * (p.D / 4) + 255) / 256;
    hipLaunchKernelGGL(rel_attn_join_kernel<T>, dim3((unsigned)(p.B * p.Hk * blocks)), dim3(256), 0, (hipStream_t)stream, p);
    OCCF_LAUNCH_CHECK();
  }
  constexpr int NT = RaType<T>::NT, KT = NT == 3 && DP > 64 ? 32 : 64;
  const size_t lds = RaFwd<T, DP, KT>::bytes(p.R);
  const long nqt = (p.Lq + 127) / 128, heads = (long)p.B * p.Hq;
  return ra_launch(rel_attn_fwd_kernel<T, DP, KT>, dim3((unsigned)(heads * nqt)), 256, lds, stream, p);
}

extern "C" long occf_rel_attn_workspace(const int64_t* geom, int dtype) {
  if (ra_check(geom, dtype)) return -1;
  int few, nsplit, chunk;
  ra_plan(geom, 0, 0, dtype, few, nsplit, chunk);        // (the parts depend on neither the mask nor the lengths)
  if (nsplit == 1) return 0;
  const long rows = geom[1] * (geom[3] / geom[4]);
  return (long)(nsplit + 1) * geom[0] * geom[4] * ((rows + 31) / 32) * 32 * (geom[5] + 2);
}

extern "C" int occf_rel_attn_fwd(const void* q, const void* k, const void* v, const void* table, const int32_t* lut,
                                 const int32_t* q_lens, const int32_t* k_lens, const int32_t* q_start, void* out, float* lse,
                                 float* workspace, long workspace_floats, const int64_t* geom, float scale, int causal,
                                 int dtype, void* stream) {
  const int bad = ra_check(geom, dtype);
  if (bad) return bad;
  if (!q || !k || !v || !table || !lut || !out || !(scale > 0.f)) return OCCF_EINVAL;
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) != 0) return OCCF_EINVAL;
  int few;
  RaParams p = ra_params(geom, scale, causal);
  ra_plan(geom, causal, k_lens != nullptr, dtype, few, p.nsplit, p.chunk);
  const long need = occf_rel_attn_workspace(geom, dtype);
  if (need > 0 && (!workspace || workspace_floats < need || ((uintptr_t)workspace & 15))) return OCCF_EINVAL;
  p.q = q; p.k = k; p.v = v; p.table = table; p.lut = lut;
  p.q_lens = q_lens; p.k_lens = k_lens; p.q_start = q_start;
  p.o = out; p.lse = lse; p.part = few && need > 0 ? workspace : nullptr;
  p.by_length = p.part && k_lens && p.B > 1 && p.B <= 512;
  p.units = p.B * (p.nsplit + p.by_length);
  RA_DISPATCH(dtype, p.D, ra_fwd, p, few, stream);
}
