// Attention with a learned relative position bias by buckets: backward (the reference's is ATen autograd through its
// attention modules, projects/mmdet3d_plugin/occformer/backbones/modules/window_attention.py:69-107).
//
//   P = exp2(t - lse),  dV = P^T dO,  dP = dO V^T,  delta_i = dO_i . O_i,  dS = P (dP - delta)
//   dQ = scale dS K,    dK = scale dS^T Q,    dT[b, h] = sum of dS over the pairs whose distance is in bucket b
//
// Two kernels, one an operand orientation, so that P and dS never leave registers and every gradient is written once, by one
// wave, in a fixed order (no atomics):
//   rel_attn_dq_kernel   a wave owns 32 queries (lane = query) and walks the keys:  S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T;
//                        also leaves delta for the other kernel and the distances' sums of dS
//   rel_attn_dkv_kernel  a wave owns 32 keys (lane = key) and walks the queries of every head that shares them:
//                        S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS
// The scores are formed twice: 7 products instead of 5, where a single pass would have to add dQ up across workgroups.
#include "rel_attn.h"
#include "../../include/occformer_hip.h"

#define RA_DLD 33               // row of the 32 x 32 tile whose diagonals are summed

// P of a lane's 16 scores: exponent base-2 t - lse, zero where the pair does not count
template <bool MASK>
__device__ __forceinline__ void ra_probs(f32x16& s, const float* bl, bool near, float far, float c, float lse, int jl, int pi,
                                         int nk, int causal) {
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int o = (r & 3) + 8 * (r >> 2);
    float t = near ? fmaf(s[r], c, bl[o] - lse) : fmaf(s[r], c, far - lse);
    if (MASK) {
      const int j = jl + o;
      if (j >= nk || (causal && j > pi)) t = -INFINITY;
    }
    s[r] = ra_exp2(t);
  }
}

template <class T, int DP, int KT, int NW>
struct RaDq {
  static constexpr int NT = RaType<T>::NT;
  static constexpr int images = NT * (2 * RaRow<DP>::bytes(KT) + RaTrans<KT>::bytes(DP));
  static size_t bytes(int R) {
    const size_t n = 2 * (size_t)R + 1 + 2 * RA_PAD;
    return images + 4 * (n + NW * n + NW * 32 * RA_DLD);
  }
};

template <class T, int DP, int KT, int NW>
__global__ void __launch_bounds__(NW * 64) rel_attn_dq_kernel(RaParams p) {
  constexpr int NT = RaType<T>::NT, KS = DP / 16, DT = DP / 32, TH = NW * 64, QW = NW * 32;
  constexpr int NB = KT * DP / 16, NU = (NB + TH - 1) / TH;
  OCCF_DYN_SMEM(smem);
  char* img_k = smem;
  char* img_v = img_k + NT * RaRow<DP>::bytes(KT);
  char* img_kt = img_v + NT * RaRow<DP>::bytes(KT);
  const int nl = 2 * p.R + 1 + 2 * RA_PAD;
  float* lut = (float*)(img_kt + NT * RaTrans<KT>::bytes(DP));
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, li = lane & 31, lk = lane >> 5;
  float* sums = lut + nl;                                // [NW][nl] sums of dS by distance
  float* dsum = sums + wave * nl;
  float* tile = sums + NW * nl + wave * 32 * RA_DLD;

  const int nqt = (p.Lq + QW - 1) / QW;
  unsigned bid = occf_xcd_remap(blockIdx.x, gridDim.x);
  const unsigned wg = bid;
  const int qt = nqt - 1 - (int)(bid % nqt);
  bid /= nqt;
  const int h = (int)(bid % p.Hq), b = (int)(bid / p.Hq);
  const int hk = h / (p.Hq / p.Hk);
  int nq, nk, start;
  ra_lengths(p, b, nq, nk, start);
  ra_fill_bias<T>(lut, p, h, tid, TH);
  for (int t = tid; t < NW * nl; t += TH) sums[t] = 0.f;

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
  if (i < p.Lq && lk == 0) p.delta[stat] = delta;

  int kend = nk;
  if (p.causal) {
    const int last = start + (qt * QW + QW < nq ? qt * QW + QW : nq);
    kend = last < kend ? (last > 0 ? last : 0) : kend;
  }
  if (qt * QW >= nq) kend = 0;
  const T* kb = (const T*)p.k + (long)b * p.ksb + (long)hk * p.ksh;
  const T* vb = (const T*)p.v + (long)b * p.vsb + (long)hk * p.vsh;

  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = ra_zero16();
  float below = 0.f, above = 0.f;                        // sums of dS at distances <= -R and >= R

  RaBlk<T> rk[NU], rv[NU];
  const int ntile = (kend + KT - 1) / KT;
  if (ntile > 0) {
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      if (NB % TH && tid + n * TH >= NB) break;
      ra_load_blk<T, DP>(rk[n], kb, p.ksl, 0, kend, p.D, tid + n * TH);
      ra_load_blk<T, DP>(rv[n], vb, p.vsl, 0, kend, p.D, tid + n * TH);
    }
  }
  for (int kt = 0; kt < ntile; ++kt) {
    const int k0 = kt * KT;
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      if (NB % TH && tid + n * TH >= NB) break;
      uint32_t w[NT][4][2];
      ra_blk_pieces(rk[n], w);
      ra_store_row<NT, DP, KT>(img_k, w, tid + n * TH);
      ra_store_trans<NT, DP, KT>(img_kt, w, tid + n * TH);
      ra_blk_pieces(rv[n], w);
      ra_store_row<NT, DP, KT>(img_v, w, tid + n * TH);
    }
    __syncthreads();
    if (kt + 1 < ntile) {
#pragma unroll
      for (int n = 0; n < NU; ++n) {
        if (NB % TH && tid + n * TH >= NB) break;
        ra_load_blk<T, DP>(rk[n], kb, p.ksl, k0 + KT, kend, p.D, tid + n * TH);
        ra_load_blk<T, DP>(rv[n], vb, p.vsl, k0 + KT, kend, p.D, tid + n * TH);
      }
    }
    if (i0 >= nq) continue;                              // wave-uniform
#pragma unroll
    for (int sub = 0; sub < KT / 32; ++sub) {
      const int j0 = k0 + sub * 32, rel0 = j0 - (start + i0);
      if (j0 >= kend || (p.causal && rel0 > 31)) continue;
      f32x16 s = ra_zero16(), dp = ra_zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = ra_mm<NT>(ra_read_row<NT, DP, KT>(img_k, sub * 32, ks, li, lk), qf[ks], s);
        dp = ra_mm<NT>(ra_read_row<NT, DP, KT>(img_v, sub * 32, ks, li, lk), of[ks], dp);
      }
      const bool near = rel0 - 31 < p.R && rel0 + 31 > -p.R;
      const float far = lut[rel0 > 0 ? 2 * p.R + RA_PAD : RA_PAD];
      const int jl = j0 + 4 * lk;
      const float* bl = lut + (near ? jl - pi + p.R + RA_PAD : 0);
      if (j0 + 32 > kend || (p.causal && rel0 + 31 > 0))
        ra_probs<true>(s, bl, near, far, p.c, lse, jl, pi, kend, p.causal);
      else
        ra_probs<false>(s, bl, near, far, p.c, lse, jl, pi, kend, p.causal);
      float ds[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] = s[r] * (dp[r] - delta);
      if (near) {
        // sums along the diagonals: lane e adds the pairs at distance rel0 + e - 31 (63 of them), in LDS of the wave's own
        RA_WAVE_SYNC();
#pragma unroll
        for (int r = 0; r < 16; ++r) tile[((r & 3) + 8 * (r >> 2) + 4 * lk) * RA_DLD + li] = ds[r];
        RA_WAVE_SYNC();
        float x = 0.f;
#pragma unroll 8
        for (int q = 0; q < 32; ++q) {
          const int row = q + lane - 31;
          if (row >= 0 && row < 32) x += tile[row * RA_DLD + q];
        }
        const int at = rel0 + lane - 31 + p.R + RA_PAD;
        if (lane < 63) dsum[at] += x;
      } else {
        float x = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) x += ds[r];
        if (rel0 > 0) above += x;
        else below += x;
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        const RaFrag<NT> df = ra_pack8<NT>(ds + s2 * 8);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          acc[dt] = ra_mm<NT>(ra_read_trans<NT, DP, KT>(img_kt, dt * 32, sub * 2 + s2, li, lk), df, acc[dt]);
      }
    }
  }
  if (i < p.Lq) {
    T* row = (T*)p.dq + orow;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = dt * 32 + 8 * g + 4 * lk;
        if (d < p.D)
          ra_store4(row + d, acc[dt][4 * g] * p.scale, acc[dt][4 * g + 1] * p.scale, acc[dt][4 * g + 2] * p.scale,
                    acc[dt][4 * g + 3] * p.scale);
      }
  }
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
  __syncthreads();
  // this workgroup's sums by clamped distance, waves in order, then the columns beyond either end
  float* part = p.part + (long)wg * (2 * p.R + 1);
  for (int t = tid; t < 2 * p.R + 1; t += TH) {
    const int lo = t == 0 ? 0 : t + RA_PAD, hi = t == 2 * p.R ? nl : t + RA_PAD + 1;
    float x = 0.f;
    for (int a = lo; a < hi; ++a)
#pragma unroll
      for (int w = 0; w < NW; ++w) x += sums[w * nl + a];
    part[t] = x;
  }
}

// dT of one head: the workgroups' sums by distance in order, then every bucket's distances in order
template <class T>
__global__ void __launch_bounds__(1024) rel_attn_dtable_kernel(RaParams p, T* dtable, int nqt) {
  OCCF_DYN_SMEM(smem);
  const int n = 2 * p.R + 1, h = blockIdx.x, tid = threadIdx.x;
  float* sum = (float*)smem;                             // [n]
  int* lut = (int*)(sum + n);                            // [n]
  for (int t = tid; t < n; t += 1024) {
    float x = 0.f;
    for (int b = 0; b < p.B; ++b) {
      const float* src = p.part + ((long)b * p.Hq + h) * nqt * n + t;
#pragma unroll 8
      for (int q = 0; q < nqt; ++q) x += src[(long)q * n];
    }
    sum[t] = x;
    lut[t] = occf_clampi(p.lut[t], p.nb - 1);
  }
  __syncthreads();
  for (int b = tid; b < p.nb; b += 1024) {
    float x = 0.f;
    for (int t = 0; t < n; ++t)
      if (lut[t] == b) x += sum[t];
    T* dst = dtable + (long)b * p.Hq + h;
    if constexpr (sizeof(T) == 4) *dst = x;
    else *dst = (T)occf_bf16_1(x);
  }
}

template <class T, int DP, int QT>
struct RaDkv {
  static constexpr int NT = RaType<T>::NT;
  static constexpr int images = 2 * NT * (RaRow<DP>::bytes(QT) + RaTrans<QT>::bytes(DP));
  static size_t bytes(int R) { return images + 4 * (2 * (size_t)R + 1 + 2 * RA_PAD + 2 * QT); }
};

template <class T, int DP, int QT, int NW>
__global__ void __launch_bounds__(NW * 64) rel_attn_dkv_kernel(RaParams p) {
  constexpr int NT = RaType<T>::NT, KS = DP / 16, DT = DP / 32, TH = NW * 64, KW = NW * 32;
  constexpr int NB = QT * DP / 16, NU = (NB + TH - 1) / TH;
  OCCF_DYN_SMEM(smem);
  char* img_q = smem;
  char* img_o = img_q + NT * RaRow<DP>::bytes(QT);
  char* img_qt = img_o + NT * RaRow<DP>::bytes(QT);
  char* img_ot = img_qt + NT * RaTrans<QT>::bytes(DP);
  float* s_lse = (float*)(img_ot + NT * RaTrans<QT>::bytes(DP));
  float* s_delta = s_lse + QT;
  float* lut = s_delta + QT;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, li = lane & 31, lk = lane >> 5;

  const int nkt = (p.Lk + KW - 1) / KW;
  unsigned bid = occf_xcd_remap(blockIdx.x, gridDim.x);
  const int kt = (int)(bid % nkt);                       // causal: the first keys have the most queries
  bid /= nkt;
  const int hk = (int)(bid % p.Hk), b = (int)(bid / p.Hk);
  const int G = p.Hq / p.Hk;
  int nq, nk, start;
  ra_lengths(p, b, nq, nk, start);

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

  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    dk[dt] = ra_zero16();
    dv[dt] = ra_zero16();
  }
  RaBlk<T> rq[NU], ro[NU];
  float nlse = 0.f, ndelta = 0.f;
  auto load = [&](int step) {
    const int h = hk * G + step / ntile, r0 = first + (step % ntile) * QT;
    const T* qb = (const T*)p.q + (long)b * p.qsb + (long)h * p.qsh;
    const T* ob = (const T*)p.dout + ((long)b * p.Lq * p.Hq + h) * p.D;
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      if (NB % TH && tid + n * TH >= NB) break;
      ra_load_blk<T, DP>(rq[n], qb, p.qsl, r0, nq, p.D, tid + n * TH);
      ra_load_blk<T, DP>(ro[n], ob, (long)p.Hq * p.D, r0, nq, p.D, tid + n * TH);
    }
    if (tid < QT) {
      const int i = r0 + tid;
      const long stat = ((long)b * p.Hq + h) * p.Lq + i;
      nlse = i < nq ? p.lse[stat] : INFINITY;
      if (nlse == -INFINITY) nlse = INFINITY;
      ndelta = i < nq ? p.delta[stat] : 0.f;
    }
  };
  const int steps = ntile * G;
  if (steps > 0) load(0);
  for (int step = 0; step < steps; ++step) {
    const int r0 = first + (step % ntile) * QT;
    __syncthreads();
    if (step % ntile == 0) ra_fill_bias<T>(lut, p, hk * G + step / ntile, tid, TH);
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      if (NB % TH && tid + n * TH >= NB) break;
      uint32_t w[NT][4][2];
      ra_blk_pieces(rq[n], w);
      ra_store_row<NT, DP, QT>(img_q, w, tid + n * TH);
      ra_store_trans<NT, DP, QT>(img_qt, w, tid + n * TH);
      ra_blk_pieces(ro[n], w);
      ra_store_row<NT, DP, QT>(img_o, w, tid + n * TH);
      ra_store_trans<NT, DP, QT>(img_ot, w, tid + n * TH);
    }
    if (tid < QT) {
      s_lse[tid] = nlse;
      s_delta[tid] = ndelta;
    }
    __syncthreads();
    if (step + 1 < steps) load(step + 1);
    if (j0 >= nk) continue;                              // wave-uniform
#pragma unroll
    for (int sub = 0; sub < QT / 32; ++sub) {
      const int i0 = r0 + sub * 32, rel0 = j0 - (start + i0);
      if (i0 >= nq || (p.causal && rel0 > 31)) continue;
      f32x16 s = ra_zero16(), dp = ra_zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = ra_mm<NT>(ra_read_row<NT, DP, QT>(img_q, sub * 32, ks, li, lk), kf[ks], s);
        dp = ra_mm<NT>(ra_read_row<NT, DP, QT>(img_o, sub * 32, ks, li, lk), vf[ks], dp);
      }
      const bool near = rel0 - 31 < p.R && rel0 + 31 > -p.R;
      const float far = lut[rel0 > 0 ? 2 * p.R + RA_PAD : RA_PAD];
      const bool mask = j0 + 32 > nk || (p.causal && rel0 + 31 > 0);
      const int il = i0 + 4 * lk;                        // rows il + (r & 3) + 8 (r >> 2)
      const float* bl = lut + (near ? j - (start + il) + p.R + RA_PAD : 32);
      float ds[16];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 ls = *(const float4*)(s_lse + sub * 32 + 8 * g + 4 * lk);
        const float4 de = *(const float4*)(s_delta + sub * 32 + 8 * g + 4 * lk);
        const float lse4[4] = {ls.x, ls.y, ls.z, ls.w}, del4[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e, o = e + 8 * g;
          float t = fmaf(s[r], p.c, (near ? bl[-o] : far) - lse4[e]);
          if (mask && (!live || (p.causal && j > start + il + o))) t = -INFINITY;
          s[r] = ra_exp2(t);
          ds[r] = s[r] * (dp[r] - del4[e]);
        }
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        float pv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) pv[e] = s[s2 * 8 + e];
        const RaFrag<NT> pf = ra_pack8<NT>(pv), df = ra_pack8<NT>(ds + s2 * 8);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          dv[dt] = ra_mm<NT>(ra_read_trans<NT, DP, QT>(img_ot, dt * 32, sub * 2 + s2, li, lk), pf, dv[dt]);
          dk[dt] = ra_mm<NT>(ra_read_trans<NT, DP, QT>(img_qt, dt * 32, sub * 2 + s2, li, lk), df, dk[dt]);
        }
      }
    }
  }
  if (j >= p.Lk) return;
  const float keep = live ? 1.f : 0.f;
  const long out = (((long)b * p.Lk + j) * p.Hk + hk) * p.D;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = dt * 32 + 8 * g + 4 * lk;
      if (d >= p.D) continue;
      const float a = p.scale * keep;
      ra_store4((T*)p.dk + out + d, dk[dt][4 * g] * a, dk[dt][4 * g + 1] * a, dk[dt][4 * g + 2] * a, dk[dt][4 * g + 3] * a);
      ra_store4((T*)p.dv + out + d, dv[dt][4 * g] * keep, dv[dt][4 * g + 1] * keep, dv[dt][4 * g + 2] * keep,
                dv[dt][4 * g + 3] * keep);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
template <class T, int DP>
static int ra_bwd(RaParams& p, void* dtable, void* stream) {
  constexpr int NW = 4, KT = RaType<T>::NT == 3 && DP > 64 ? 32 : 64, QT = RaType<T>::NT == 3 ? 32 : 64;
  const int nqt = (p.Lq + NW * 32 - 1) / (NW * 32), nkt = (p.Lk + NW * 32 - 1) / (NW * 32);
  int rc = ra_launch(rel_attn_dq_kernel<T, DP, KT, NW>, dim3((unsigned)((long)p.B * p.Hq * nqt)), NW * 64,
                     RaDq<T, DP, KT, NW>::bytes(p.R), stream, p);
  if (rc) return rc;
  rc = ra_launch(rel_attn_dkv_kernel<T, DP, QT, NW>, dim3((unsigned)((long)p.B * p.Hk * nkt)), NW * 64,
                 RaDkv<T, DP, QT>::bytes(p.R), stream, p);
  if (rc) return rc;
  hipLaunchKernelGGL(rel_attn_dtable_kernel<T>, dim3(p.Hq), dim3(1024), 8 * (2 * (size_t)p.R + 1), (hipStream_t)stream, p,
                     (T*)dtable, nqt);
  OCCF_LAUNCH_CHECK();
}

extern "C" long occf_rel_attn_bwd_workspace(const int64_t* geom, int dtype) {
  if (ra_check(geom, dtype)) return -1;
  const long B = geom[0], Lq = geom[1], Hq = geom[3], R = geom[7];
  return B * Hq * Lq + B * Hq * ((Lq + 127) / 128) * (2 * R + 1);
}

extern "C" int occf_rel_attn_bwd(const void* q, const void* k, const void* v, const void* table, const int32_t* lut,
                                 const int32_t* q_lens, const int32_t* k_lens, const int32_t* q_start, const void* out,
                                 const float* lse, const void* dout, void* dq, void* dk, void* dv, void* dtable,
                                 float* workspace, long workspace_floats, const int64_t* geom, float scale, int causal,
                                 int dtype, void* stream) {
  const int bad = ra_check(geom, dtype);
  if (bad) return bad;
  if (!q || !k || !v || !table || !lut || !out || !lse || !dout || !dq || !dk || !dv || !dtable || !workspace || !(scale > 0.f))
    return OCCF_EINVAL;
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk |
        (uintptr_t)dv) & 15) != 0)
    return OCCF_EINVAL;
  if (workspace_floats < occf_rel_attn_bwd_workspace(geom, dtype)) return OCCF_EINVAL;
  RaParams p = ra_params(geom, scale, causal);
  p.q = q; p.k = k; p.v = v; p.table = table; p.lut = lut;
  p.q_lens = q_lens; p.k_lens = k_lens; p.q_start = q_start;
  p.out = out; p.dout = dout; p.lse = (float*)lse;
  p.dq = dq; p.dk = dk; p.dv = dv;
  p.delta = workspace;
  p.part = workspace + (long)p.B * p.Hq * p.Lq;
  RA_DISPATCH(dtype, p.D, ra_bwd, p, dtable, stream);
}
