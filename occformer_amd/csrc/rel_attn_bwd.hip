// Attention with a learned relative position bias by buckets: backward (the reference's is ATen autograd through its
// attention modules, projects/mmdet3d_plugin/occformer/backbones/modules/window_attention.py:69-107).
//
//   P = exp2(t - lse),  dV = P^T dO,  dP = dO V^T,  delta_i = dO_i . O_i,  dS = P (dP - delta)
//   dQ = scale dS K,    dK = scale dS^T Q,    dT[b, h] = sum of dS over the pairs whose distance is in bucket b
//
// Two kernels, one an operand orientation, so that P and dS never leave registers and every sum has a fixed order (no atomics):
//   rel_attn_dq_kernel   a wave owns 32 queries (lane = query) and walks the keys:  S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T
//   rel_attn_dkv_kernel  a wave owns 32 keys (lane = key) and walks the queries of every head that shares them:
//                        S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS, and the distances' sums of dS
// The scores are formed twice: 7 products instead of 5, where a single pass would have to add dQ up across workgroups.
// -delta (in the second kernel, for bf16, -lse / c too) is the accumulators' first value: no instruction a score.
//
// delta: a row of dS sums to zero, but <dO, O> of an O rounded to bf16 (whose P was rounded too) is off by a few 2^-9, and the
// bias' gradient, sums of dS that nearly cancel, shows it (3.5e-3 of error where its own rounding is 1.7e-3).  The row sums of
// the dS so formed ARE that error (P sums to one), so the first kernel adds them to the delta that the second one reads, and
// takes (row sum) x (P K) off its own dQ: one product more, bf16 only; an fp32 O leaves nothing to correct in dQ.
//
// 2 x 4096 causal bf16 rows, 16 / 4 heads of 64: 141 and 198 us, 970 and 690 TFLOP/s of four products each.  Matrix pipes, vector
// instructions and LDS are busy 42, 43 and 27 % of the first, 26, 32 and 33 % of the second, whose operands come as rows and as columns
// and whose diagonals' sums go through the LDS between barriers.  2 x 1000 fp32 rows, 8 heads of 24: 29 and 39 us, short walks of
// 256 and 512 workgroups.  (Comparisons below are of short runs, in which the card has not reached its clock: up to a fifth more.)
//
// Both walks are cut into `splits` where whole ones would not fill the card; rel_attn_finish_kernel adds the parts up in order.
#include "rel_attn.h"
#include "../../include/occformer_hip.h"

// The 32 x 32 tile whose diagonals are summed: rows of 64 floats of which the last 32 stay zero, as do 32 before the first, so
// that a lane's walk down its diagonal needs no test (32 reads at constant offsets).  fp32 with more than 64 columns has room for
// half a tile beside its operand images, and sums it in two goes.
template <class T, int DP> struct RaDiag {
  static constexpr int ROWS = RaType<T>::NT == 3 && DP > 64 ? 16 : 32, LD = 64, FRONT = 32, floats = FRONT + ROWS * LD;
};

struct RaBwd {
  RaParams a;
  void* dtable;
  float *eps, *dq_part, *pk_part, *dk_part, *dv_part, *tab_part;
  int qsplit, ksplit;            // parts of the keys a query's walk is cut into; parts of the queries a key's
};

template <class T, int DP, int KT>
struct RaDq {
  static constexpr int tile = 2 * RaType<T>::NT * RaRow<DP>::bytes(KT);                  // K and V
  static size_t bytes(int R) { return tile + 4 * (2 * (size_t)R + 1 + 2 * RA_PAD); }
};

template <class T, int DP, int KT, int NW, int NP>
__global__ void __launch_bounds__(NW * 64, RA_WAVES_PER_SIMD(T, DP)) rel_attn_dq_kernel(RaBwd g) {
  const RaParams& p = g.a;
  constexpr int NT = RaType<T>::NT, KS = DP / 16, DT = DP / 32, TH = NW * 64, QW = NW * 32;
  constexpr bool PK = NT == 1;
  OCCF_DYN_SMEM(smem);
  float* lut = (float*)(smem + RaDq<T, DP, KT>::tile);
  const int tid = threadIdx.x, wave = occf_wave_uniform(tid >> 6), lane = tid & 63, li = lane & 31, lk = lane >> 5;

  const int nqt = (p.Lq + QW - 1) / QW;
  int qt, bh;
  ra_order(p, blockIdx.x, nqt, p.B * p.Hq * g.qsplit, qt, bh);
  qt = nqt - 1 - qt;
  const int split = bh % g.qsplit;
  bh /= g.qsplit;
  const int h = bh % p.Hq, b = bh / p.Hq;
  const int hk = h / (p.Hq / p.Hk);
  int nq, nk, start;
  ra_lengths(p, b, nq, nk, start);
  ra_fill_bias<T>(lut, p, h, tid, TH);
  float far_below, far_above;
  ra_far_bias<T>(p, h, far_below, far_above);

  const int i0 = qt * QW + wave * 32, i = i0 + li, pi = start + i;
  const bool live = i < nq;
  const int ic = occf_clampi(i, p.Lq - 1);
  const T* qrow = (const T*)p.q + (long)b * p.qsb + (long)ic * p.qsl + (long)h * p.qsh;
  const long orow = (((long)b * p.Lq + ic) * p.Hq + h) * p.D;
  RaFrag<NT> qf[KS], of[KS];
  float delta = 0.f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int d = ks * 16 + lk * 8;
    const bool ok = live && d < p.D;
    qf[ks] = ra_row_frag<T>(qrow + (d < p.D ? d : 0), ok);
    of[ks] = ra_row_frag<T>((const T*)p.dout + orow + (d < p.D ? d : 0), ok);
    if (ok) {
      const T *x = (const T*)p.out + orow + d, *y = (const T*)p.dout + orow + d;
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = fmaf(ra_to_float(x[e]), ra_to_float(y[e]), delta);
    }
  }
  delta += __shfl_xor(delta, 32);
  const long stat = ((long)b * p.Hq + h) * p.Lq + ic;
  float lse = live ? p.lse[stat] : INFINITY;
  if (lse == -INFINITY) lse = INFINITY;                  // no key: P = 0
  const bool some = lse != INFINITY;
  const f32x16 dp_first = ra_splat16(-delta);

  int kend = nk;
  if (p.causal) {
    const int last = start + (qt * QW + QW < nq ? qt * QW + QW : nq);
    kend = last < kend ? (last > 0 ? last : 0) : kend;
  }
  if (qt * QW >= nq) kend = 0;
  const T* kb = (const T*)p.k + (long)b * p.ksb + (long)hk * p.ksh;
  const T* vb = (const T*)p.v + (long)b * p.vsb + (long)hk * p.vsh;

  f32x16 acc[DT], pk[PK ? DT : 1];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = ra_zero16();
#pragma unroll
  for (int dt = 0; dt < (PK ? DT : 1); ++dt) pk[dt] = ra_zero16();
  float eps = 0.f;

  RaTileRegs<T, DP, KT, TH> rk, rv;
  rk.place(p.ksl, p.D, tid);
  rv.place(p.vsl, p.D, tid);
  const int ntile = (kend + KT - 1) / KT;
  const int t0 = (int)((unsigned)(ntile * split) / (unsigned)g.qsplit), t1 = (int)((unsigned)(ntile * (split + 1)) / (unsigned)g.qsplit);
  const auto load = [&](int k0) {
    rk.load(kb + k0 * p.ksl, p.ksl, kend - k0, p.D);
    rv.load(vb + k0 * p.vsl, p.vsl, kend - k0, p.D);
  };
  const char *img_k = smem, *img_v = smem + NT * RaRow<DP>::bytes(KT);
  load(t0 * KT);
  RA_WAIT_LOADS();
  for (int kt = t0; kt < t1; ++kt) {
    const int k0 = kt * KT;
    __syncthreads();
    rk.store(smem, tid);
    rv.store(smem + NT * RaRow<DP>::bytes(KT), tid);
    __syncthreads();
    load(k0 + KT);
    if (i0 >= nq) continue;                              // wave-uniform
#pragma unroll 1
    for (int sub = 0; sub < KT / 32; ++sub) {
      const int j0 = k0 + sub * 32, rel0 = j0 - (start + i0);
      if (j0 >= kend || (p.causal && rel0 > 31)) continue;
      f32x16 s = ra_zero16(), dp = dp_first;
      RA_PRIO(1);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = ra_mm<NT>(ra_read_row<NT, DP, KT>(img_k, sub * 32, ks, li, lk), qf[ks], s);
        dp = ra_mm<NT>(ra_read_row<NT, DP, KT>(img_v, sub * 32, ks, li, lk), of[ks], dp);
      }
      RA_PRIO(0);
      const bool near = rel0 - 31 < p.R && rel0 + 31 > -p.R;
      const int jl = j0 + 4 * lk;
      float ce, be;
      ra_bias_mask<1>(s, lut + (near ? jl - pi + p.R + RA_PAD : 0), near, rel0 > 0 ? far_above : far_below,
                      j0 + 32 > kend || (p.causal && rel0 + 31 > 0), p.c, ce, be,
                      [&](int o) { return jl + o >= kend || (p.causal && jl + o > pi); });
      be -= lse;
      float ds[16], pv[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        pv[r] = ra_exp2(fmaf(s[r], ce, be));
        ds[r] = pv[r] * dp[r];
        eps += ds[r];
      }
      RA_PRIO(1);
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const RaFrag<NP> df = ra_pack8<NP>(ds + s2 * 8);
        const RaFrag<NT> pf = ra_pack8<NT>(pv + s2 * 8);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const RaFrag<NT> kt_f = ra_read_trans<NT, DP, KT>(img_k, dt * 32, sub * 2 + s2, lane);
          acc[dt] = ra_mm(kt_f, df, acc[dt]);
          if (PK) pk[dt] = ra_mm<NT>(kt_f, pf, pk[dt]);
        }
      }
      RA_PRIO(0);
    }
  }
  eps += __shfl_xor(eps, 32);
  if (i >= p.Lq) return;
  if (!some) {                                           // went along with their tile: 0 times an infinite key is no zero
    delta = eps = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = ra_zero16();
#pragma unroll
    for (int dt = 0; dt < (PK ? DT : 1); ++dt) pk[dt] = ra_zero16();
  }
  if (lk == 0) {
    if (split == 0) p.delta[stat] = g.qsplit > 1 ? delta : delta + eps;
    if (g.qsplit > 1) g.eps[(long)split * p.B * p.Hq * p.Lq + stat] = eps;      // rel_attn_finish_kernel adds these to delta
  }
  const long part = (long)split * p.B * p.Lq * p.Hq * p.D + orow;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = dt * 32 + 8 * q + 4 * lk;
      if (d >= p.D) continue;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = acc[dt][4 * q + e];
      if (g.qsplit > 1) {
        ra_store4(g.dq_part + part + d, x[0], x[1], x[2], x[3]);
        if (PK) ra_store4(g.pk_part + part + d, pk[dt][4 * q], pk[dt][4 * q + 1], pk[dt][4 * q + 2], pk[dt][4 * q + 3]);
        continue;
      }
      if (PK) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = fmaf(-eps, pk[dt][4 * q + e], x[e]);
      }
      ra_store4((T*)p.dq + orow + d, x[0] * p.scale, x[1] * p.scale, x[2] * p.scale, x[3] * p.scale);
    }
}

template <class T, int DP, int QT, int NW>
struct RaDkv {
  static constexpr int images = 2 * RaType<T>::NT * RaRow<DP>::bytes(QT);                // Q and dO
  static constexpr int tile = images + 2 * QT * 4;                                       // and the rows' statistics
  // two images where they are small: a tile then costs one barrier, the next one is stored while others still read this one
  // (232 instead of 240 us at 2 x 4096 causal rows, 16 / 4 heads of 64)
  static constexpr int NBUF = tile <= 20 * 1024 ? 2 : 1;
  static size_t bytes(int R) {
    const size_t nl = 2 * (size_t)R + 1 + 2 * RA_PAD;
    return NBUF * tile + 4 * ((NW + 1) * nl + NW * RaDiag<T, DP>::floats) + nl;
  }
};

template <class T, int DP, int QT, int NW, int NP>
__global__ void __launch_bounds__(NW * 64, RA_WAVES_PER_SIMD(T, DP)) rel_attn_dkv_kernel(RaBwd g) {
  const RaParams& p = g.a;
  typedef RaDkv<T, DP, QT, NW> L;
  constexpr int NT = RaType<T>::NT, KS = DP / 16, DT = DP / 32, TH = NW * 64, KW = NW * 32, NBUF = L::NBUF;
  // -lse / c as the scores' first value rounds every partial sum at its size (12 / c = 40 at 1000 keys): 1e-6 of P, not for fp32
  constexpr bool LSE_FIRST = NT == 1;
  OCCF_DYN_SMEM(smem);
  float* tiles = (float*)(smem + NBUF * L::tile);
  float* lut = tiles + NW * RaDiag<T, DP>::floats;
  const int nl = 2 * p.R + 1 + 2 * RA_PAD;
  float* sums = lut + nl;                                // [NW][nl] sums of dS by distance
  const int tid = threadIdx.x, wave = occf_wave_uniform(tid >> 6), lane = tid & 63, li = lane & 31, lk = lane >> 5;
  float* dsum = sums + wave * nl;
  float* tile = tiles + wave * RaDiag<T, DP>::floats + RaDiag<T, DP>::FRONT;
  uint8_t* ids = (uint8_t*)(sums + NW * nl);             // bucket of every distance

  const int nkt = (p.Lk + KW - 1) / KW, G = p.Hq / p.Hk;
  int kt, bh;
  ra_order(p, blockIdx.x, nkt, p.B * p.Hk * g.ksplit, kt, bh);         // the first keys are seen by the most queries
  const int split = bh % g.ksplit;
  bh /= g.ksplit;
  const int hk = bh % p.Hk, b = bh / p.Hk;
  int nq, nk, start;
  ra_lengths(p, b, nq, nk, start);
  if (p.causal) {                                        // keys behind the last query: nobody sees them, nor are they looked at
    const int last = start + nq;
    nk = last < nk ? (last > 0 ? last : 0) : nk;
  }

  const int j0 = kt * KW + wave * 32, j = j0 + li;
  const bool live = j < nk;
  const int jc = occf_clampi(j, p.Lk - 1);
  const T* krow = (const T*)p.k + (long)b * p.ksb + (long)jc * p.ksl + (long)hk * p.ksh;
  const T* vrow = (const T*)p.v + (long)b * p.vsb + (long)jc * p.vsl + (long)hk * p.vsh;
  RaFrag<NT> kf[KS], vf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int d = ks * 16 + lk * 8;
    const bool ok = live && d < p.D;
    kf[ks] = ra_row_frag<T>(krow + (d < p.D ? d : 0), ok);
    vf[ks] = ra_row_frag<T>(vrow + (d < p.D ? d : 0), ok);
  }
  // first query tile with a query at or behind the workgroup's first key
  int first = 0;
  if (p.causal) {
    const int at = kt * KW - start;
    first = at > 0 ? at / QT * QT : 0;
  }
  const int ntile = kt * KW >= nk || first >= nq ? 0 : (nq - first + QT - 1) / QT;
  // steps: the query tiles of every head of the group, in order; this workgroup's share of them
  const unsigned steps = (unsigned)(ntile * G);
  const int t0 = (int)(steps * split / (unsigned)g.ksplit), t1 = (int)(steps * (split + 1) / (unsigned)g.ksplit);
  float far_below = 0.f, far_above = 0.f;                // the head's biases at distances <= -R and >= R
  const int hg0 = t0 < t1 ? t0 / ntile : 0;
  ra_fill_bias<T>(lut, p, hk * G + hg0, tid, TH);
  ra_far_bias<T>(p, hk * G + hg0, far_below, far_above);
  for (int t = tid; t < nl; t += TH) ids[t] = (uint8_t)occf_clampi(p.lut[occf_clampi(t - RA_PAD, 2 * p.R)], p.nb - 1);
  for (int t = tid; t < NW * RaDiag<T, DP>::floats / 4; t += TH) ra_store4(tiles + 4 * t, 0.f, 0.f, 0.f, 0.f);
  float* tab = g.tab_part + ((((long)b * p.Hk + hk) * g.ksplit + split) * nkt + kt) * G * p.nb;       // [G][nb]

  for (int t = tid; t < NW * nl; t += TH) sums[t] = 0.f;
  // heads that this share does not touch
  for (int t = tid; t < G * p.nb; t += TH) {
    const int hg = t / p.nb;
    if (t0 >= t1 || hg < t0 / ntile || hg > (t1 - 1) / ntile) tab[t] = 0.f;
  }

  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    dk[dt] = ra_zero16();
    dv[dt] = ra_zero16();
  }
  float below = 0.f, above = 0.f;                        // sums of dS at distances <= -R and >= R
  RaTileRegs<T, DP, QT, TH> rq, ro;
  const long osl = (long)p.Hq * p.D;
  rq.place(p.qsl, p.D, tid);
  ro.place(osl, p.D, tid);
  // the next tile's rows, and on QT lanes their statistics, all looked at only when the tile is stored: a value that is used
  // where it is loaded would make the workgroup wait for it in every step
  float nlse = 0.f, ndelta = 0.f;
  const long nstat = (long)p.Hq * p.Lq;
  const occf_bbuf lse_buf = occf_make_bbuf(p.lse + b * nstat, (uint32_t)nstat * 4u);
  const occf_bbuf delta_buf = occf_make_bbuf(p.delta + b * nstat, (uint32_t)nstat * 4u);
  int hg = hg0, at = t0 - hg * ntile;                                    // head of the group and query tile of a step
  int lstep = t0, lhg = hg, lat = at;                                    // ... of the next load
  int nrow = 0, nend = 0;                                                // the loaded tile's first query, and behind its last
  const auto load = [&]() {
    const bool more = lstep < t1;                                        // (else: no rows)
    const int h = hk * G + (more ? lhg : 0), r0 = more ? first + lat * QT : 0;
    nrow = r0;
    nend = more ? nq : 0;
    rq.load((const T*)p.q + (long)b * p.qsb + (long)h * p.qsh + r0 * p.qsl, p.qsl, nend - r0, p.D);
    ro.load((const T*)p.dout + ((long)b * p.Lq * p.Hq + h) * p.D + r0 * osl, osl, nend - r0, p.D);
    const uint32_t stat = tid < QT && r0 + tid < nend ? ((uint32_t)h * (uint32_t)p.Lq + (uint32_t)(r0 + tid)) * 4u : OCCF_BUF_OOB;
    nlse = ra_buf4(lse_buf, stat);
    ndelta = ra_buf4(delta_buf, stat);
    ++lstep;
    if (++lat == ntile) {
      lat = 0;
      ++lhg;
    }
  };
  // s_lse, s_delta: first values of the accumulators' rows
  const auto store = [&](int buf) {
    char* to = smem + buf * L::tile;
    rq.store(to, tid);
    ro.store(to + NT * RaRow<DP>::bytes(QT), tid);
    float *s_lse = (float*)(to + L::images), *s_delta = s_lse + QT;
    if (tid < QT) {
      // rows that do not count or see no key: P = 0 (the former are hidden as well: a row of zeros times an infinite key is NaN)
      const bool row = nrow + tid < nend;
      s_lse[tid] = !row || nlse == -INFINITY ? -INFINITY : LSE_FIRST ? -nlse / p.c : -nlse;
      s_delta[tid] = -ndelta;
    }
  };
  load();
  RA_WAIT_LOADS();
  if (NBUF == 2) {
    store(0);
    load();
  }
  for (int step = t0; step < t1; ++step, ++at) {
    if (at == ntile) {
      at = 0;
      ++hg;
    }
    const int r0 = first + at * QT;
    __syncthreads();
    if (step > t0 && at == 0) {
      ra_fill_bias<T>(lut, p, hk * G + hg, tid, TH);
      ra_far_bias<T>(p, hk * G + hg, far_below, far_above);
      if (NBUF == 2) __syncthreads();
    }
    if (NBUF == 1) {
      store(0);
      __syncthreads();
      load();
    } else {
      store((step + 1 - t0) & 1);
      load();
    }
    const char* img_q = smem + (NBUF == 2 ? (step - t0) & 1 : 0) * L::tile;
    const char* img_o = img_q + NT * RaRow<DP>::bytes(QT);
    const float *s_lse = (const float*)(img_q + L::images), *s_delta = s_lse + QT;
#pragma unroll 1
    for (int sub = 0; sub < QT / 32; ++sub) {
      const int i0 = r0 + sub * 32, rel0 = j0 - (start + i0);
      if (j0 >= nk || i0 >= nq || (p.causal && rel0 > 31)) continue;      // wave-uniform
      f32x16 s, dp;
      float off[LSE_FIRST ? 1 : 16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 x = *(const float4*)(s_lse + sub * 32 + 8 * q + 4 * lk);
        const float4 y = *(const float4*)(s_delta + sub * 32 + 8 * q + 4 * lk);
        s[4 * q] = x.x; s[4 * q + 1] = x.y; s[4 * q + 2] = x.z; s[4 * q + 3] = x.w;
        if (!LSE_FIRST) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            off[LSE_FIRST ? 0 : 4 * q + e] = s[4 * q + e];
            s[4 * q + e] = 0.f;
          }
        }
        dp[4 * q] = y.x; dp[4 * q + 1] = y.y; dp[4 * q + 2] = y.z; dp[4 * q + 3] = y.w;
      }
      RA_PRIO(1);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = ra_mm<NT>(ra_read_row<NT, DP, QT>(img_q, sub * 32, ks, li, lk), kf[ks], s);
        dp = ra_mm<NT>(ra_read_row<NT, DP, QT>(img_o, sub * 32, ks, li, lk), vf[ks], dp);
      }
      RA_PRIO(0);
      const bool near = rel0 - 31 < p.R && rel0 + 31 > -p.R;
      const int pl = start + i0 + 4 * lk;                // position of row 0 of this lane
      // rows [lo, lo + n) of it count: the queries before the last, causal: at or behind the key
      const int lo = p.causal && j > pl ? j - pl : 0, end = live ? start + nq - pl : 0;
      const unsigned n = end > lo ? end - lo : 0;
      float ce, be;
      ra_bias_mask<-1>(s, lut + (near ? j - pl + p.R + RA_PAD : 32), near, rel0 > 0 ? far_above : far_below,
                       j0 + 32 > nk || i0 + 32 > nq || (p.causal && rel0 + 31 > 0), p.c, ce, be,
                       [&](int o) { return (unsigned)(o - lo) >= n; });
      float ds[16], pv[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        pv[r] = ra_exp2(fmaf(s[r], ce, LSE_FIRST ? be : be + off[LSE_FIRST ? 0 : r]));
        ds[r] = pv[r] * dp[r];
      }
      if (near) {
        // sums along the diagonals: lane e adds the pairs at distance rel0 + e - 31 (63 of them), in LDS of the wave's own
        constexpr int DR = RaDiag<T, DP>::ROWS, DL = RaDiag<T, DP>::LD;
        float y[2] = {0.f, 0.f};
        const float* dg = tile + lane - 31;
#pragma unroll
        for (int hv = 0; hv < 32 / DR; ++hv) {
          RA_WAVE_SYNC();
#pragma unroll
          for (int r = 0; r < DR / 2; ++r) tile[((r & 3) + 8 * (r >> 2) + 4 * lk) * DL + li] = ds[DR / 2 * hv + r];
          RA_WAVE_SYNC();
#pragma unroll
          for (int q = 0; q < DR; ++q) y[q & 1] += dg[q * (DL + 1) + DR * hv];
        }
        const float x = y[0] + y[1];
        if (lane < 63) dsum[rel0 + lane - 31 + p.R + RA_PAD] += x;
      } else {
        float x = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) x += ds[r];
        if (rel0 > 0) above += x;
        else below += x;
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const RaFrag<NP> pf = ra_pack8<NP>(pv + s2 * 8), df = ra_pack8<NP>(ds + s2 * 8);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          dv[dt] = ra_mm(ra_read_trans<NT, DP, QT>(img_o, dt * 32, sub * 2 + s2, lane), pf, dv[dt]);
          dk[dt] = ra_mm(ra_read_trans<NT, DP, QT>(img_q, dt * 32, sub * 2 + s2, lane), df, dk[dt]);
        }
      }
    }
    if (step + 1 == t1 || at + 1 == ntile) {
      // a head is done: its distances' sums, waves in order, then the buckets', distances in order
#pragma unroll
      for (int mm = 32; mm > 0; mm >>= 1) {
        below += __shfl_xor(below, mm);
        above += __shfl_xor(above, mm);
      }
      RA_WAVE_SYNC();
      if (lane == 0) {
        dsum[0] += below;
        dsum[nl - 1] += above;
      }
      below = above = 0.f;
      __syncthreads();
      for (int t = tid; t < nl; t += TH) {
        float x = sums[t];
#pragma unroll
        for (int w = 1; w < NW; ++w) {
          x += sums[w * nl + t];
          sums[w * nl + t] = 0.f;
        }
        sums[t] = x;
      }
      __syncthreads();
      // `tl` threads a bucket walk every tl-th distance (the columns beyond either end count as the end)
      int nb2 = 4;
      while (nb2 < p.nb) nb2 <<= 1;
      const int tl = TH / nb2, bk = tid / tl, r = tid % tl;
      float x = 0.f;
      if (bk < p.nb)
#pragma unroll 4
        for (int t = r; t < nl; t += tl) x += ids[t] == bk ? sums[t] : 0.f;
      for (int mm = 1; mm < tl; mm <<= 1) x += __shfl_xor(x, mm);
      if (bk < p.nb && r == 0) tab[hg * p.nb + bk] = x;
      __syncthreads();
      for (int t = tid; t < nl; t += TH) sums[t] = 0.f;
    }
  }
  if (j >= p.Lk) return;
  const long out = (((long)b * p.Lk + j) * p.Hk + hk) * p.D;
  const long part = (long)split * p.B * p.Lk * p.Hk * p.D + out;
  if (!live) {                                           // keys that do not count
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dk[dt] = dv[dt] = ra_zero16();
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = dt * 32 + 8 * q + 4 * lk;
      if (d >= p.D) continue;
      const f32x16 &x = dk[dt], &y = dv[dt];
      if (g.ksplit > 1) {
        ra_store4(g.dk_part + part + d, x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
        ra_store4(g.dv_part + part + d, y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
      } else {
        ra_store4((T*)p.dk + out + d, x[4 * q] * p.scale, x[4 * q + 1] * p.scale, x[4 * q + 2] * p.scale, x[4 * q + 3] * p.scale);
        ra_store4((T*)p.dv + out + d, y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
      }
    }
}

// The parts in order, a stream (12.4 us for 75 MB, four parts of 2 x 4096 x 4 heads of 64 keys and values).  Behind the first
// kernel, where its walk was cut: dq (four columns a thread), and a row's first thread completes its delta.  Behind the second:
// the bias' gradient on Hq workgroups, then dk and dv where that walk was cut.
template <class T>
__global__ void __launch_bounds__(256) rel_attn_finish_kernel(RaBwd g, int nkt, int dq) {
  const RaParams& p = g.a;
  const int tid = threadIdx.x;
  int blk = blockIdx.x;
  if (!dq && blk < p.Hq) {
    __shared__ float acc[256];
    const int G = p.Hq / p.Hk, hk = blk / G, hg = blk % G;
    int nb2 = 1;
    while (nb2 < p.nb) nb2 <<= 1;
    const int b = tid % nb2, r = tid / nb2, lanes = 256 / nb2;
    const int rows = g.ksplit * nkt;
    float x = 0.f;
    if (b < p.nb)
      for (int s = 0; s < p.B; ++s) {
        const float* src = g.tab_part + (((long)s * p.Hk + hk) * rows * G + hg) * p.nb + b;
#pragma unroll 4
        for (int q = r; q < rows; q += lanes) x += src[(long)q * G * p.nb];
      }
    acc[tid] = x;
    __syncthreads();
    if (r == 0 && b < p.nb) {
      x = 0.f;
      for (int q = 0; q < lanes; ++q) x += acc[q * nb2 + b];
      T* dst = (T*)g.dtable + (long)b * p.Hq + blk;
      if constexpr (sizeof(T) == 4) *dst = x;
      else *dst = (T)occf_bf16_1(x);
    }
    return;
  }
  if (!dq) blk -= p.Hq;
  const long at = ((long)blk * 256 + tid) * 4;
  const long n = dq ? (long)p.B * p.Lq * p.Hq * p.D : (long)p.B * p.Lk * p.Hk * p.D;
  if (at >= n) return;
  const int splits = dq ? g.qsplit : g.ksplit;
  const float *pa = dq ? g.dq_part : g.dk_part, *pb = dq ? g.pk_part : g.dv_part;
  const bool second = !dq || RaType<T>::NT == 1;
  float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) {
    const float4 a = *(const float4*)(pa + s * n + at);
    x[0] += a.x; x[1] += a.y; x[2] += a.z; x[3] += a.w;
    if (second) {
      const float4 c = *(const float4*)(pb + s * n + at);
      y[0] += c.x; y[1] += c.y; y[2] += c.z; y[3] += c.w;
    }
  }
  if (dq) {
    const long row = at / p.D;                           // (b Lq + i) Hq + h
    const int h = (int)(row % p.Hq);
    const long bi = row / p.Hq;
    const long stat = (bi / p.Lq * p.Hq + h) * p.Lq + bi % p.Lq;
    float eps = 0.f;
    for (int s = 0; s < splits; ++s) eps += g.eps[(long)s * p.B * p.Hq * p.Lq + stat];
    if (at == row * p.D) p.delta[stat] += eps;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (second ? fmaf(-eps, y[e], x[e]) : x[e]) * p.scale;
    ra_store4((T*)p.dq + at, x[0], x[1], x[2], x[3]);
  } else {
    ra_store4((T*)p.dk + at, x[0] * p.scale, x[1] * p.scale, x[2] * p.scale, x[3] * p.scale);
    ra_store4((T*)p.dv + at, y[0], y[1], y[2], y[3]);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// How often the walks are cut, 128 rows or more a part.  A key's: until there are as many workgroups as the card's registers hold
// (one or two a compute unit, by type and head dim; beyond that is a second round: 120 instead of 101 us for the whole
// backward at 2048 rows, 4 heads of 128), twice as many of a causal walk's unequal key tiles (a quarter off that kernel's time at
// 2 x 4096, 4 key heads of 64).  A query's: one a compute unit, its parts of two matrices cost more than the second one brings (79 instead
// of 90 us at 3 x 777, 12 heads of 64).
static void ra_bwd_plan(const int64_t* g, int causal, int dtype, int& qsplit, int& ksplit) {
  const long B = g[0], Lq = g[1], Lk = g[2], Hq = g[3], Hk = g[4];
  const long slots = 256 * (dtype == 0 ? RA_WAVES_PER_SIMD(float, g[5]) : RA_WAVES_PER_SIMD(ra_bf16, g[5]));
  const long wq = B * Hq * ((Lq + 127) / 128), wk = B * Hk * ((Lk + 127) / 128);
  const long mq = (Lk + 127) / 128, mk = (Hq / Hk) * ((Lq + 127) / 128);
  const auto cut = [](long want, long most) { return (int)(want < 1 ? 1 : want > most ? most : want); };
  qsplit = cut(cut(256 / wq, mq), 8);
  ksplit = cut(cut((causal ? 2 : 1) * slots / wk, mk), 16);
}

struct RaBwdSizes { long delta, eps, dq, dk, tab; };
static RaBwdSizes ra_bwd_sizes(const int64_t* g, int qsplit, int ksplit) {
  const long B = g[0], Lq = g[1], Lk = g[2], Hq = g[3], Hk = g[4], D = g[5], nb = g[6];
  RaBwdSizes s;
  const auto up = [](long n) { return (n + 63) / 64 * 64; };             // parts start on 256 bytes
  s.delta = up(B * Hq * Lq);
  s.eps = qsplit > 1 ? up(B * Hq * Lq * qsplit) : 0;
  s.dq = qsplit > 1 ? up(B * Lq * Hq * D * qsplit) : 0;
  s.dk = ksplit > 1 ? up(B * Lk * Hk * D * ksplit) : 0;
  s.tab = up(B * Hq * ksplit * ((Lk + 127) / 128) * nb);
  return s;
}

template <class T, int DP, int NP>
static int ra_bwd_run(const RaBwd& g, void* stream) {
  constexpr int NW = 4, KT = RaType<T>::NT == 3 && DP > 64 ? 32 : 64, QT = RaType<T>::NT == 3 ? 32 : 64;
  const RaParams& p = g.a;
  const long nqt = (p.Lq + NW * 32 - 1) / (NW * 32), nkt = (p.Lk + NW * 32 - 1) / (NW * 32);
  int rc = ra_launch(rel_attn_dq_kernel<T, DP, KT, NW, NP>, dim3((unsigned)(p.B * p.Hq * nqt * g.qsplit)), NW * 64,
                     RaDq<T, DP, KT>::bytes(p.R), stream, g);
  if (rc) return rc;
  const auto blocks = [](long n) { return (unsigned)((n / 4 + 255) / 256); };
  if (g.qsplit > 1) {
    hipLaunchKernelGGL(rel_attn_finish_kernel<T>, dim3(blocks((long)p.B * p.Lq * p.Hq * p.D)), dim3(256), 0, (hipStream_t)stream,
                       g, (int)nkt, 1);
    rc = (int)hipGetLastError();
    if (rc) return rc;
  }
  rc = ra_launch(rel_attn_dkv_kernel<T, DP, QT, NW, NP>, dim3((unsigned)(p.B * p.Hk * nkt * g.ksplit)), NW * 64,
                 RaDkv<T, DP, QT, NW>::bytes(p.R), stream, g);
  if (rc) return rc;
  hipLaunchKernelGGL(rel_attn_finish_kernel<T>, dim3(p.Hq + (g.ksplit > 1 ? blocks((long)p.B * p.Lk * p.Hk * p.D) : 0)), dim3(256), 0,
                     (hipStream_t)stream, g, (int)nkt, 0);
  OCCF_LAUNCH_CHECK();
}

// bf16: P and dS go into their products rounded to bf16, or as two bf16 pieces (2^-16) where no walk is longer than 512.  The
// rounding makes dq, dk and dv about sqrt(2) times as far off as their own rounding alone, and in a short walk, where a few values
// make up a sum, up to 1.7 times.  Two pieces are one more instruction a product: 45.9 instead of 44.7 us at 2 x 384, 12 heads of
// 64, but 92.8 instead of 86.1 at 3 x 777 and 546 instead of 459 at 2 x 4096 (forward included, causal, 16 / 4 heads).
template <class T, int DP>
static int ra_bwd(const RaBwd& g, void* stream) {
  if constexpr (RaType<T>::NT == 3) return ra_bwd_run<T, DP, 3>(g, stream);
  else return g.a.Lq <= 512 && g.a.Lk <= 512 ? ra_bwd_run<T, DP, 2>(g, stream) : ra_bwd_run<T, DP, 1>(g, stream);
}

// rows of dO lie Hq D elements apart: 64 of them within 2 GiB, as ra_check has it for q, k and v (heads of q that are one head
// repeated may be many and lie close)
static int ra_bwd_check(const int64_t* g, int dtype) {
  const int bad = ra_check(g, dtype);
  return bad ? bad : g[3] * g[5] >= (1L << 22) ? OCCF_ESHAPE : 0;
}

extern "C" long occf_rel_attn_bwd_workspace(const int64_t* geom, int causal, int dtype) {
  if (ra_bwd_check(geom, dtype)) return -1;
  int qs, ks;
  ra_bwd_plan(geom, causal, dtype, qs, ks);
  const RaBwdSizes s = ra_bwd_sizes(geom, qs, ks);
  return s.delta + s.eps + s.dq * (dtype == 1 ? 2 : 1) + s.dk * 2 + s.tab;
}

extern "C" int occf_rel_attn_bwd(const void* q, const void* k, const void* v, const void* table, const int32_t* lut,
                                 const int32_t* q_lens, const int32_t* k_lens, const int32_t* q_start, const void* out,
                                 const float* lse, const void* dout, void* dq, void* dk, void* dv, void* dtable,
                                 float* workspace, long workspace_floats, const int64_t* geom, float scale, int causal,
                                 int dtype, void* stream) {
  const int bad = ra_bwd_check(geom, dtype);
  if (bad) return bad;
  if (!q || !k || !v || !table || !lut || !out || !lse || !dout || !dq || !dk || !dv || !dtable || !workspace || !(scale > 0.f))
    return OCCF_EINVAL;
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)dout | (uintptr_t)workspace | (uintptr_t)dq | (uintptr_t)dk |
        (uintptr_t)dv) & 15) != 0)
    return OCCF_EINVAL;
  if (workspace_floats < occf_rel_attn_bwd_workspace(geom, causal, dtype)) return OCCF_EINVAL;
  RaBwd g = {};
  g.a = ra_params(geom, scale, causal);
  RaParams& p = g.a;
  p.q = q; p.k = k; p.v = v; p.table = table; p.lut = lut;
  p.q_lens = q_lens; p.k_lens = k_lens; p.q_start = q_start;
  p.out = out; p.dout = dout; p.lse = (float*)lse;
  p.dq = dq; p.dk = dk; p.dv = dv;
  g.dtable = dtable;
  ra_bwd_plan(geom, causal, dtype, g.qsplit, g.ksplit);
  const RaBwdSizes s = ra_bwd_sizes(geom, g.qsplit, g.ksplit);
  p.delta = workspace;
  g.eps = p.delta + s.delta;
  g.dq_part = g.eps + s.eps;
  g.pk_part = g.dq_part + s.dq;
  g.dk_part = g.pk_part + (dtype == 1 ? s.dq : 0);
  g.dv_part = g.dk_part + s.dk;
  g.tab_part = g.dv_part + s.dk;
  RA_DISPATCH(dtype, p.D, ra_bwd, g, stream);
}
