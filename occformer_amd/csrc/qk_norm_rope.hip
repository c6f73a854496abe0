// Norms of queries and keys for each head with the position rotation in the same pass, and their backward.
//
//   a row x (one token, one head, D values), weight w:   r = 1 / sqrt(mean(x^2) + eps),  y = x r w
//   pairs (a, b) of y's first `rot` columns:             (a cos - b sin, b cos + a sin),  angle row = position of the token
//   backward:  dy = turn dz back;  dw += dy x r;  g = dy w;  dx = r (g - x r mean(g x r))
//
// The reference adds absolute position codes to whole tokens (LearnedPositionalEncoding / SinePositionalEncoding3D of its
// occupancy decoder, projects/mmdet3d_plugin/occformer/mask2former/positional_encodings/); this turns every head's rows.
//
// One pass, bound by the memory stream: a row is VEC pairs a lane, its D / 2 / VEC lanes (rounded up to a power of two) sum
// the squares by shuffles, so that a row is read once and written once; the angles' cosines and sines come from a table made
// in 64 bits (a far position's angle loses digits in 32) whose row is shared by the heads of a token.
// Forward, 2 x 8192 tokens of 32 + 8 bf16 heads of 128: 68.5 us, 5.0 TB/s.  4 x 4095 tokens of 16 + 4 bf16 heads of 64:
// 21 us, backward 28.6 us, 4.4 TB/s, and 3.9 us for the weights' sums of at most 512 workgroups a side, in a fixed order.
#include "occf_common.h"
#include "../../include/occformer_hip.h"

typedef uint16_t qn_bf16;

struct QnSide {                     // queries or keys
  const void *x, *dz, *w;
  void* out;                        // z, or dx
  long sb, sl, sh;                  // element strides of x: batch, token, head
  int H, blocks;
};
struct QnParams {
  QnSide s[2];
  const float *cos, *sin;
  const int32_t* pos;
  float* part;                      // backward: [blocks of q and k][D] sums of dw
  long pos_b;                       // positions: elements a batch entry (0 = shared)
  int B, L, D, half, P, axes, cut1, cut2, lpr;      // half = rotated pairs; axis of pair c: 0 below cut1, 1 below cut2, else 2
  float eps;
};

template <class T, int V> struct alignas(sizeof(T) * V) QnVec { T e[V]; };

__device__ __forceinline__ float qn_f(float x) { return x; }
__device__ __forceinline__ float qn_f(qn_bf16 x) { return occf_u2f((uint32_t)x << 16); }
__device__ __forceinline__ void qn_put(float& t, float x) { t = x; }
__device__ __forceinline__ void qn_put(qn_bf16& t, float x) { t = (qn_bf16)occf_bf16_1(x); }

// V pairs of a row: columns ca .. and cb .. (two halves), or 2 V neighbouring columns (interleaved)
template <class T, int V, bool INTER>
__device__ __forceinline__ void qn_load(const T* p, int ca, int cb, float (&a)[V], float (&b)[V]) {
  if (INTER) {
    const QnVec<T, 2 * V> x = *(const QnVec<T, 2 * V>*)(p + ca);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      a[e] = qn_f(x.e[2 * e]);
      b[e] = qn_f(x.e[2 * e + 1]);
    }
  } else {
    const QnVec<T, V> x = *(const QnVec<T, V>*)(p + ca), y = *(const QnVec<T, V>*)(p + cb);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      a[e] = qn_f(x.e[e]);
      b[e] = qn_f(y.e[e]);
    }
  }
}
template <class T, int V, bool INTER>
__device__ __forceinline__ void qn_store(T* p, int ca, int cb, const float (&a)[V], const float (&b)[V]) {
  if (INTER) {
    QnVec<T, 2 * V> x;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      qn_put(x.e[2 * e], a[e]);
      qn_put(x.e[2 * e + 1], b[e]);
    }
    *(QnVec<T, 2 * V>*)(p + ca) = x;
  } else {
    QnVec<T, V> x, y;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      qn_put(x.e[e], a[e]);
      qn_put(y.e[e], b[e]);
    }
    *(QnVec<T, V>*)(p + ca) = x;
    *(QnVec<T, V>*)(p + cb) = y;
  }
}

// cosines and sines of the V pairs from pc at token (b, l); a position outside the table turns its row into NaN
template <int V>
__device__ __forceinline__ void qn_angles(const QnParams& p, int b, int l, int pc, float (&c)[V], float (&s)[V]) {
  if (pc >= p.half) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      c[e] = 1.f;
      s[e] = 0.f;
    }
    return;
  }
  const int32_t* pp = p.pos + b * p.pos_b + (long)l * p.axes;
  if (p.axes == 1) {
    const int at = p.pos ? pp[0] : l;
    const long o = (long)occf_clampi(at, p.P - 1) * p.half + pc;
    const QnVec<float, V> x = *(const QnVec<float, V>*)(p.cos + o), y = *(const QnVec<float, V>*)(p.sin + o);
    const bool ok = at >= 0 && at < p.P;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      c[e] = ok ? x.e[e] : NAN;
      s[e] = y.e[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int at = pp[pc + e < p.cut1 ? 0 : (pc + e < p.cut2 ? 1 : 2)];
      const long o = (long)occf_clampi(at, p.P - 1) * p.half + pc + e;
      c[e] = at >= 0 && at < p.P ? p.cos[o] : NAN;
      s[e] = p.sin[o];
    }
  }
}

__device__ __forceinline__ float qn_sum(float x, int lpr) {
  for (int m = lpr >> 1; m > 0; m >>= 1) x += __shfl_xor(x, m);
  return x;
}

template <class T, int V, bool INTER, bool BWD>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(QnParams p) {
  const int which = (int)blockIdx.x >= p.s[0].blocks;
  const QnSide& s = p.s[which];
  const int blk = (int)blockIdx.x - (which ? p.s[0].blocks : 0);
  const int lpr = p.lpr, rpb = 256 / lpr;                 // lanes a row, rows a workgroup and step
  const int lane = threadIdx.x % lpr, slot = threadIdx.x / lpr;
  const int pc = lane * V, pairs = p.D / 2;
  const bool on = pc < pairs, turned = pc < p.half;       // (a load's pairs are turned or not together)
  const int tail = pairs - p.half;                        // pairs of the columns that are not turned
  const int ca = INTER ? 2 * pc : (pc < p.half ? pc : 2 * p.half + pc - p.half);
  const int cb = INTER ? 0 : (pc < p.half ? pc + p.half : ca + tail);

  float wa[V], wb[V], da[V], db[V];
#pragma unroll
  for (int e = 0; e < V; ++e) wa[e] = wb[e] = da[e] = db[e] = 0.f;
  if (on) qn_load<T, V, INTER>((const T*)s.w, ca, cb, wa, wb);

  const long rows = (long)p.B * p.L * s.H;
  const float inv_d = 1.0f / (float)p.D;
  for (long r0 = (long)blk * rpb; r0 < rows; r0 += (long)s.blocks * rpb) {
    const long row = r0 + slot;
    const bool live = on && row < rows;
    float a[V], b[V], c[V], sn[V];
#pragma unroll
    for (int e = 0; e < V; ++e) a[e] = b[e] = 0.f;
    if (live) {
      const unsigned tok = (unsigned)row / (unsigned)s.H, h = (unsigned)row - tok * (unsigned)s.H;
      const unsigned bi = tok / (unsigned)p.L, l = tok - bi * (unsigned)p.L;
      qn_load<T, V, INTER>((const T*)s.x + (long)bi * s.sb + (long)l * s.sl + (long)h * s.sh, ca, cb, a, b);
      qn_angles<V>(p, (int)bi, (int)l, pc, c, sn);
    }
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) q = fmaf(a[e], a[e], fmaf(b[e], b[e], q));
    q = qn_sum(q, lpr);
    const float rs = 1.0f / sqrtf(fmaf(q, inv_d, p.eps));
    if (!BWD) {
      if (live) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float ya = a[e] * rs * wa[e], yb = b[e] * rs * wb[e];
          a[e] = turned ? fmaf(ya, c[e], -(yb * sn[e])) : ya;       // (0 times a partner's NaN is no zero)
          b[e] = turned ? fmaf(yb, c[e], ya * sn[e]) : yb;
        }
        qn_store<T, V, INTER>((T*)s.out + row * p.D, ca, cb, a, b);
      }
    } else {
      float ga[V], gb[V];
#pragma unroll
      for (int e = 0; e < V; ++e) ga[e] = gb[e] = 0.f;
      float dot = 0.f;
      if (live) {
        qn_load<T, V, INTER>((const T*)s.dz + row * p.D, ca, cb, ga, gb);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float ya = turned ? fmaf(ga[e], c[e], gb[e] * sn[e]) : ga[e];
          const float yb = turned ? fmaf(gb[e], c[e], -(ga[e] * sn[e])) : gb[e];
          a[e] *= rs;
          b[e] *= rs;
          da[e] = fmaf(ya, a[e], da[e]);
          db[e] = fmaf(yb, b[e], db[e]);
          ga[e] = ya * wa[e];
          gb[e] = yb * wb[e];
          dot = fmaf(ga[e], a[e], fmaf(gb[e], b[e], dot));
        }
      }
      dot = qn_sum(dot, lpr) * inv_d;
      if (live) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          ga[e] = rs * fmaf(-a[e], dot, ga[e]);
          gb[e] = rs * fmaf(-b[e], dot, gb[e]);
        }
        qn_store<T, V, INTER>((T*)s.out + row * p.D, ca, cb, ga, gb);
      }
    }
  }
  if (BWD) {
    // sums of the workgroup's rows in slot order
    __shared__ float acc[256 * 16];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      acc[(threadIdx.x * V + e) * 2] = da[e];
      acc[(threadIdx.x * V + e) * 2 + 1] = db[e];
    }
    __syncthreads();
    for (int t = threadIdx.x; t < p.D; t += 256) {
      // column t -> (pair, which of the two)
      int pr, second;
      if (INTER) {
        pr = t >> 1;
        second = t & 1;
      } else if (t < 2 * p.half) {
        second = t >= p.half;
        pr = second ? t - p.half : t;
      } else {
        const int o = t - 2 * p.half;
        second = o >= tail;
        pr = p.half + (second ? o - tail : o);
      }
      // four sums side by side, then in pairs: a quarter of the roundings at the size of the whole
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < rpb; k += 4)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += acc[(((k + e) * lpr) * V + pr) * 2 + second];
      p.part[(long)blockIdx.x * p.D + t] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
  }
}

// dw of queries and keys from the workgroups' sums: 8 columns a workgroup, 32 rows of sums side by side
template <class T>
__global__ void __launch_bounds__(256) qk_norm_rope_dw_kernel(const float* __restrict__ part, T* __restrict__ dwq,
                                                              T* __restrict__ dwk, int nq, int nk, int D) {
  __shared__ float acc[32][8];
  const int cols = (D + 7) / 8;
  const int which = (int)blockIdx.x >= cols;
  const int c = ((int)blockIdx.x - (which ? cols : 0)) * 8 + (threadIdx.x & 7), r = threadIdx.x >> 3;
  const int n = which ? nk : nq;
  const float* src = part + (which ? (long)nq * D : 0);
  float sum = 0.f;
  if (c < D)
#pragma unroll 8
    for (int i = r; i < n; i += 32) sum += src[(long)i * D + c];
  acc[r][threadIdx.x & 7] = sum;
  __syncthreads();
  if (r == 0 && c < D) {
    float t[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < 32; i += 4)
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] += acc[i + e][threadIdx.x & 7];
    qn_put((which ? dwk : dwq)[c], (t[0] + t[1]) + (t[2] + t[3]));
  }
}

// geom = [B, L, Hq, Hk (0: no keys), D, rotated columns, table rows, axes, cut1, cut2, positions a batch entry (0 shared),
//         q strides b l h, k strides b l h]
static int qn_setup(QnParams& p, const void* q, const void* k, const void* qw, const void* kw, const float* cos,
                    const float* sin, const int32_t* pos, const int64_t* g, float eps, int interleaved, int dtype, bool bwd,
                    int& V) {
  if (!g || !q || !qw || (dtype != 0 && dtype != 1)) return OCCF_EINVAL;
  const long B = g[0], L = g[1], Hq = g[2], Hk = g[3], D = g[4], rot = g[5], P = g[6], axes = g[7];
  if (B <= 0 || L <= 0 || Hq <= 0 || Hk < 0 || D < 2 || D > 128 || D % 2 || rot < 0 || rot > D || rot % 2) return OCCF_ESHAPE;
  if (Hk && (!k || !kw)) return OCCF_EINVAL;
  if (rot && (!cos || !sin || P <= 0 || axes < 1 || axes > 3 || (axes > 1 && !pos))) return OCCF_EINVAL;
  if (rot && axes > 1 && (g[8] < 1 || g[9] < g[8] || (axes == 2 && g[9] < rot / 2))) return OCCF_EINVAL;   // no column of a third axis
  if (B * L * (Hq > Hk ? Hq : Hk) >= 2147483647L) return OCCF_ESHAPE;
  if (P > 2147483647L || g[8] > D || g[9] > D) return OCCF_ESHAPE;
  const int esize = dtype == 0 ? 4 : 2, pairs = (int)D / 2, half = (int)rot / 2;
  // the widest vectors that the columns, the strides and the addresses allow: 16 bytes a load, else half that, else single pairs
  uintptr_t align = (uintptr_t)q | (uintptr_t)k | (uintptr_t)qw | (uintptr_t)kw;
  for (int s = 11; s < (Hk ? 17 : 14); ++s) align |= (uintptr_t)(g[s] * esize);
  const int wide = 16 / esize;                                    // columns of 16 bytes
  V = 1;
  for (int v = interleaved ? wide / 2 : wide; v > 1; v >>= 1) {
    const unsigned bytes = (unsigned)(v * esize * (interleaved ? 2 : 1));
    if (half % v == 0 && (pairs - half) % v == 0 && align % bytes == 0 && ((uintptr_t)cos | (uintptr_t)sin) % (v * 4) == 0 &&
        D * esize % bytes == 0) {
      V = v;
      break;
    }
  }
  if (interleaved && V == 1 && align % (2 * esize)) return OCCF_EINVAL;      // a pair is one load
  int lpr = 1;
  while (lpr * V < pairs) lpr <<= 1;
  p.B = (int)B; p.L = (int)L; p.D = (int)D; p.half = half; p.P = (int)P; p.axes = rot ? (int)axes : 1;
  p.cut1 = (int)g[8]; p.cut2 = (int)g[9]; p.pos_b = g[10]; p.lpr = lpr; p.eps = eps;
  p.cos = cos; p.sin = sin; p.pos = pos;
  p.s[0] = QnSide{q, nullptr, qw, nullptr, g[11], g[12], g[13], (int)Hq, 0};
  p.s[1] = QnSide{k, nullptr, kw, nullptr, g[14], g[15], g[16], (int)Hk, 0};
  const long rpb = 256 / lpr;
  for (int i = 0; i < 2; ++i) {
    const long n = (B * L * (i ? Hk : Hq) + rpb - 1) / rpb, most = bwd ? 512 : 8192;
    p.s[i].blocks = (int)(n < most ? n : most);
  }
  return 0;
}

template <class T, bool BWD>
static void qn_run(const QnParams& p, int V, int interleaved, void* stream) {
  const dim3 grid(p.s[0].blocks + p.s[1].blocks);
#define QN_GO(v, i) hipLaunchKernelGGL((qk_norm_rope_kernel<T, v, i, BWD>), grid, dim3(256), 0, (hipStream_t)stream, p)
  if (interleaved) {
    if (sizeof(T) == 2 && V == 4) QN_GO(sizeof(T) == 2 ? 4 : 2, true);
    else if (V == 2) QN_GO(2, true);
    else QN_GO(1, true);
  } else {
    if (sizeof(T) == 2 && V == 8) QN_GO(sizeof(T) == 2 ? 8 : 4, false);
    else if (V == 4) QN_GO(4, false);
    else if (V == 2) QN_GO(2, false);
    else QN_GO(1, false);
  }
#undef QN_GO
}

extern "C" int occf_qk_norm_rope_fwd(const void* q, const void* k, const void* q_weight, const void* k_weight,
                                     const float* cos, const float* sin, const int32_t* positions, void* q_out,
                                     void* k_out, const int64_t* geom, float eps, int interleaved, int dtype, void* stream) {
  QnParams p = {};
  int V;
  const int rc = qn_setup(p, q, k, q_weight, k_weight, cos, sin, positions, geom, eps, interleaved, dtype, false, V);
  if (rc) return rc;
  if (!q_out || (geom[3] && !k_out) || (((uintptr_t)q_out | (uintptr_t)k_out) & 15)) return OCCF_EINVAL;
  p.s[0].out = q_out;
  p.s[1].out = k_out;
  if (dtype == 0) qn_run<float, false>(p, V, interleaved, stream);
  else qn_run<qn_bf16, false>(p, V, interleaved, stream);
  OCCF_LAUNCH_CHECK();
}

extern "C" long occf_qk_norm_rope_bwd_workspace(int head_dim) { return 1024L * head_dim; }

extern "C" int occf_qk_norm_rope_bwd(const void* q, const void* k, const void* q_weight, const void* k_weight,
                                     const float* cos, const float* sin, const int32_t* positions, const void* dq_out,
                                     const void* dk_out, void* dq, void* dk, void* dq_weight, void* dk_weight,
                                     float* workspace, const int64_t* geom, float eps, int interleaved, int dtype,
                                     void* stream) {
  QnParams p = {};
  int V;
  const int rc = qn_setup(p, q, k, q_weight, k_weight, cos, sin, positions, geom, eps, interleaved, dtype, true, V);
  if (rc) return rc;
  const bool keys = geom[3] != 0;
  if (!dq_out || !dq || !dq_weight || !workspace || (keys && (!dk_out || !dk || !dk_weight))) return OCCF_EINVAL;
  if (((uintptr_t)dq_out | (uintptr_t)dq | (uintptr_t)dk_out | (uintptr_t)dk) & 15) return OCCF_EINVAL;
  p.s[0].dz = dq_out; p.s[0].out = dq;
  p.s[1].dz = dk_out; p.s[1].out = dk;
  p.part = workspace;
  if (dtype == 0) qn_run<float, true>(p, V, interleaved, stream);
  else qn_run<qn_bf16, true>(p, V, interleaved, stream);
  const dim3 grid(((p.D + 7) / 8) * (keys ? 2 : 1));
  if (dtype == 0)
    hipLaunchKernelGGL(qk_norm_rope_dw_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, workspace, (float*)dq_weight,
                       (float*)dk_weight, p.s[0].blocks, p.s[1].blocks, p.D);
  else
    hipLaunchKernelGGL(qk_norm_rope_dw_kernel<qn_bf16>, grid, dim3(256), 0, (hipStream_t)stream, workspace,
                       (qn_bf16*)dq_weight, (qn_bf16*)dk_weight, p.s[0].blocks, p.s[1].blocks, p.D);
  OCCF_LAUNCH_CHECK();
}
