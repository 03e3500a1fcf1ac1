// Group norm + activation (+ shortcut) on channels-last rows, forward and backward.
//
//   xh = (x - mean) rstd,  u = gamma xh + beta,  out = act(u) + res          mean, rstd over the HW * C/groups values of (image, group)
//   du = dout act'(u),  dbeta = sum du,  dgamma = sum du xh,  v = gamma du
//   dx = rstd (v - mean(v) - xh mean(v xh))                                  means over the same (image, group)
//
// Both directions are HBM streams around one reduction, and the reduction separates them into two launches: the first leaves one partial
// per (image, chunk of rows) in the workspace, the second joins the partials of its image in a fixed order in its prologue (a few KB out of
// L2) and streams.  A thread owns one vector of channels for the whole launch and walks down the rows, as in the BatchNorm kernels.
//
// The variance is never formed as E[x^2] - E[x]^2: a thread sums deviations from its own first value, (count, mean, M2) triples are joined
// by Chan's formula, and the means of the triples are kept as distances from the first value of their (image, group): neither a mean of
// thousands of spreads nor one huge value costs digits.
#include "common.h"

namespace {

constexpr int GN_MAXC = 4096;    // channels (LDS: two floats each)

// V channels of one row as fp32: the 16-byte vector of Vec<T>, or (V == 1) one element at any alignment
template <typename T, int V> struct Lane {
  static DEVINL void load(const T* p, float (&f)[V]) { Vec<T>::load(p, f); }
  static DEVINL void store(T* p, const float (&f)[V]) { Vec<T>::store(p, f); }
};
template <typename T> struct Lane<T, 1> {
  static DEVINL void load(const T* p, float (&f)[1]) { f[0] = ActT<T>::ld(p); }
  static DEVINL void store(T* p, const float (&f)[1]) { ActT<T>::st(p, f[0]); }
};

struct GnP {
  const void* x;
  const void* dout;
  const void* res;
  void* out;           // forward: out; backward: dx
  const float* gamma;
  const float* beta;
  float* stats;        // [N][G][2]
  float2* gpart;       // [N][chunks][G]: forward (mean - origin, M2), backward (sum v, sum v xh)
  float* origin;       // [N][G]: the forward's origins, kept because the second launch may write over x
  float2* cpart;       // [N][chunks][C]: backward (sum du, sum du xh)
  float* dgamma;
  float* dbeta;
  int N, HW, C, G, cg, act;
  int x_ld, d_ld, r_ld, o_ld;
  int chunks, rows;    // row chunks per image, rows per chunk
  int acc_dx, acc_par;
  float eps;
};

// lanes per group for the joins below: a power of two <= 64 with lanes * G <= 256 where that is possible
DEVINL int join_lanes(int G) {
  int l = 64;
  while (l > 1 && l * G > 256) l >>= 1;
  return l;
}
template <typename A> DEVINL A lane_sum(A v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// ------------------------------------------------------------------------------------------------ forward
// the value from which the means of (image, group) are counted
template <typename T> DEVINL float gn_origin(const GnP& p, int n, int g) {
  return ActT<T>::ld((const T*)p.x + (size_t)n * p.HW * p.x_ld + (size_t)g * p.cg);
}

// (mean - origin, M2) of every group over the rows of one chunk
template <typename T, int V> __global__ __launch_bounds__(256) void gn_stats_kernel(const GnP p) {
  extern __shared__ float2 chan[];             // [C] (mean - origin, M2) of one channel over the chunk
  __shared__ float2 red[256 * V];
  const int n = blockIdx.x / p.chunks, j = blockIdx.x % p.chunks;
  const int r0 = j * p.rows, nr = min(p.HW - r0, p.rows);
  const int cv = p.C / V, cols = min(cv, 256), rpb = 256 / cols;
  const int tcol = threadIdx.x % cols, trow = threadIdx.x / cols;
  const T* base = (const T*)p.x + ((size_t)n * p.HW + r0) * p.x_ld;
  for (int cb = 0; cb < cv; cb += cols) {
    const int col = cb + tcol;
    if (col < cv && trow < rpb) {
      const T* px = base + (size_t)col * V;
      float k[V], s[V], q[V], f[V];
#pragma unroll
      for (int e = 0; e < V; ++e) k[e] = s[e] = q[e] = 0.f;
      if (trow < nr) Lane<T, V>::load(px + (size_t)trow * p.x_ld, k);
      int cnt = trow < nr ? 1 : 0;
#pragma unroll 4
      for (int r = trow + rpb; r < nr; r += rpb) {
        Lane<T, V>::load(px + (size_t)r * p.x_ld, f);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = f[e] - k[e];
          s[e] += d;
          q[e] = fmaf(d, d, q[e]);
        }
        ++cnt;
      }
      const float inv = cnt > 0 ? 1.0f / (float)cnt : 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float m2 = q[e] - s[e] * s[e] * inv;
        const float from = k[e] - gn_origin<T>(p, n, (col * V + e) / p.cg);
        red[(trow * cols + tcol) * V + e] = make_float2(from + s[e] * inv, m2 < 0.f ? 0.f : m2);   // (a NaN passes)
      }
    }
    __syncthreads();
    const int nch = min(cols, cv - cb) * V;
    for (int t = threadIdx.x; t < nch; t += 256) {
      float cnt = 0.f, mean = 0.f, m2 = 0.f;
      for (int w = 0; w < rpb && w < nr; ++w) {
        const float2 o = red[w * cols * V + t];
        const float nb = (float)((nr - w + rpb - 1) / rpb), tot = cnt + nb, d = o.x - mean;
        m2 += o.y + (cnt > 0.f ? d * d * (cnt * nb / tot) : 0.f);
        mean += d * (nb / tot);
        cnt = tot;
      }
      chan[(size_t)cb * V + t] = make_float2(mean, m2);
    }
    __syncthreads();
  }
  // channels -> groups: equal counts, so the group's mean is the mean of means
  const int L = join_lanes(p.G), gl = threadIdx.x % L, gstep = 256 / L;
  for (int g0 = 0; g0 < p.G; g0 += gstep) {
    const int g = g0 + threadIdx.x / L;
    const bool on = g < p.G;
    float sm = 0.f;
    const float first = on ? chan[g * p.cg].x : 0.f;      // the spread of the means about one of them: no digits lost to their size
    if (on) for (int c = gl; c < p.cg; c += L) sm += chan[g * p.cg + c].x - first;
    const float mean = first + lane_sum(sm, L) / (float)p.cg;
    float m2 = 0.f;
    if (on)
      for (int c = gl; c < p.cg; c += L) {
        const float2 o = chan[g * p.cg + c];
        const float d = o.x - mean;
        m2 += o.y + d * d * (float)nr;
      }
    m2 = lane_sum(m2, L);
    if (on && gl == 0) {
      p.gpart[((size_t)n * p.chunks + j) * p.G + g] = make_float2(mean, m2);
      if (j == 0) p.origin[(size_t)n * p.G + g] = gn_origin<T>(p, n, g);
    }
  }
}

// joins the chunk partials of image n: gm[2 g], gm[2 g + 1] = mean, rstd
DEVINL void gn_join_stats(const GnP& p, int n, float* gm) {
  const int L = join_lanes(p.G), gl = threadIdx.x % L, gstep = 256 / L;
  const float2* part = p.gpart + (size_t)n * p.chunks * p.G;
  const double total = (double)p.HW * p.cg;
  for (int g0 = 0; g0 < p.G; g0 += gstep) {
    const int g = g0 + threadIdx.x / L;
    const bool on = g < p.G;
    double sm = 0.0;
    if (on)
      for (int j = gl; j < p.chunks; j += L) sm += (double)part[(size_t)j * p.G + g].x * (double)min(p.HW - j * p.rows, p.rows);
    const double mean = lane_sum(sm, L) / (double)p.HW;
    double m2 = 0.0;
    if (on)
      for (int j = gl; j < p.chunks; j += L) {
        const float2 o = part[(size_t)j * p.G + g];
        const double d = (double)o.x - mean;
        m2 += (double)o.y + d * d * ((double)min(p.HW - j * p.rows, p.rows) * p.cg);
      }
    m2 = lane_sum(m2, L);
    if (on && gl == 0) {
      gm[2 * g] = (float)(mean + (double)p.origin[(size_t)n * p.G + g]);
      gm[2 * g + 1] = (float)(1.0 / sqrt(m2 / total + (double)p.eps));
    }
  }
}

template <typename T, int V, int ACTC> __global__ __launch_bounds__(256) void gn_apply_kernel(const GnP p) {
  extern __shared__ float gm[];                // [G][2]
  const int n = blockIdx.x / p.chunks, j = blockIdx.x % p.chunks;
  const int r0 = j * p.rows, nr = min(p.HW - r0, p.rows);
  const int act = ACTC >= 0 ? ACTC : p.act;
  gn_join_stats(p, n, gm);
  __syncthreads();
  if (j == 0)
    for (int t = threadIdx.x; t < 2 * p.G; t += 256) p.stats[(size_t)n * 2 * p.G + t] = gm[t];
  const int cv = p.C / V, cols = min(cv, 256), rpb = 256 / cols;
  const int tcol = threadIdx.x % cols, trow = threadIdx.x / cols;
  if (trow >= rpb) return;
  const size_t row0 = (size_t)n * p.HW + r0;
  for (int col = tcol; col < cv; col += cols) {
    float mu[V], a[V], b[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = col * V + e, g = c / p.cg;
      mu[e] = gm[2 * g];
      a[e] = gm[2 * g + 1] * (p.gamma ? p.gamma[c] : 1.f);
      b[e] = p.beta ? p.beta[c] : 0.f;
    }
    const T* px = (const T*)p.x + row0 * p.x_ld + (size_t)col * V;
    const T* pr = p.res ? (const T*)p.res + row0 * p.r_ld + (size_t)col * V : nullptr;
    T* po = (T*)p.out + row0 * p.o_ld + (size_t)col * V;
#pragma unroll 4
    for (int r = trow; r < nr; r += rpb) {
      float f[V], t[V];
      Lane<T, V>::load(px + (size_t)r * p.x_ld, f);
      if (pr) Lane<T, V>::load(pr + (size_t)r * p.r_ld, t);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[e] = actf<Vec<T>::precise>(fmaf(f[e] - mu[e], a[e], b[e]), act);
        if (pr) f[e] += t[e];
      }
      Lane<T, V>::store(po + (size_t)r * p.o_ld, f);
    }
  }
}

// ------------------------------------------------------------------------------------------------ backward
// per chunk: (sum du, sum du xh) of every channel, and (sum v, sum v xh) of every group
template <typename T, int V, int ACTC> __global__ __launch_bounds__(256) void gn_bwd_sums_kernel(const GnP p) {
  extern __shared__ float2 chan[];
  __shared__ float2 red[256 * V];
  const int n = blockIdx.x / p.chunks, j = blockIdx.x % p.chunks;
  const int r0 = j * p.rows, nr = min(p.HW - r0, p.rows);
  const int act = ACTC >= 0 ? ACTC : p.act;
  const int cv = p.C / V, cols = min(cv, 256), rpb = 256 / cols;
  const int tcol = threadIdx.x % cols, trow = threadIdx.x / cols;
  const size_t row0 = (size_t)n * p.HW + r0;
  const float* st = p.stats + (size_t)n * 2 * p.G;
  float2* cp = p.cpart + ((size_t)n * p.chunks + j) * p.C;
  for (int cb = 0; cb < cv; cb += cols) {
    const int col = cb + tcol;
    if (col < cv && trow < rpb) {
      float mu[V], rs[V], ga[V], be[V], sa[V], sb[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int c = col * V + e, g = c / p.cg;
        mu[e] = st[2 * g];
        rs[e] = st[2 * g + 1];
        ga[e] = p.gamma ? p.gamma[c] : 1.f;
        be[e] = p.beta ? p.beta[c] : 0.f;
        sa[e] = sb[e] = 0.f;
      }
      const T* px = (const T*)p.x + row0 * p.x_ld + (size_t)col * V;
      const T* pd = (const T*)p.dout + row0 * p.d_ld + (size_t)col * V;
#pragma unroll 2
      for (int r = trow; r < nr; r += rpb) {
        float f[V], d[V];
        Lane<T, V>::load(px + (size_t)r * p.x_ld, f);
        Lane<T, V>::load(pd + (size_t)r * p.d_ld, d);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float xh = (f[e] - mu[e]) * rs[e];
          const float du = d[e] * act_grad<Vec<T>::precise>(fmaf(ga[e], xh, be[e]), act);
          sa[e] += du;
          sb[e] = fmaf(du, xh, sb[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) red[(trow * cols + tcol) * V + e] = make_float2(sa[e], sb[e]);
    }
    __syncthreads();
    const int nch = min(cols, cv - cb) * V;
    for (int t = threadIdx.x; t < nch; t += 256) {
      float a = 0.f, b = 0.f;
      for (int w = 0; w < rpb && w < nr; ++w) {
        const float2 o = red[w * cols * V + t];
        a += o.x;
        b += o.y;
      }
      const int c = cb * V + t;
      chan[c] = make_float2(a, b);
      cp[c] = make_float2(a, b);
    }
    __syncthreads();
  }
  const int L = join_lanes(p.G), gl = threadIdx.x % L, gstep = 256 / L;
  for (int g0 = 0; g0 < p.G; g0 += gstep) {
    const int g = g0 + threadIdx.x / L;
    float a = 0.f, b = 0.f;
    if (g < p.G)
      for (int c = g * p.cg + gl; c < (g + 1) * p.cg; c += L) {
        const float ga = p.gamma ? p.gamma[c] : 1.f;
        a = fmaf(ga, chan[c].x, a);
        b = fmaf(ga, chan[c].y, b);
      }
    a = lane_sum(a, L);
    b = lane_sum(b, L);
    if (g < p.G && gl == 0) p.gpart[((size_t)n * p.chunks + j) * p.G + g] = make_float2(a, b);
  }
}

constexpr int GN_PC = 32;    // channels per parameter workgroup

// workgroups [0, npar): dgamma / dbeta of GN_PC channels, summed over all chunks in a fixed order; the others: dx of one chunk of rows
template <typename T, int V, int ACTC> __global__ __launch_bounds__(256) void gn_bwd_dx_kernel(const GnP p, const int npar) {
  extern __shared__ float gm[];                // [G][2]: the two means of the group
  const int act = ACTC >= 0 ? ACTC : p.act;
  if ((int)blockIdx.x < npar) {
    const int c = blockIdx.x * GN_PC + threadIdx.x % GN_PC, lane = threadIdx.x / GN_PC;
    double a = 0.0, b = 0.0;
    const size_t parts = (size_t)p.N * p.chunks;
    if (c < p.C)
      for (size_t i = lane; i < parts; i += 256 / GN_PC) {
        const float2 o = p.cpart[i * p.C + c];
        a += (double)o.x;
        b += (double)o.y;
      }
    __shared__ double da[256], db[256];
    da[threadIdx.x] = a;
    db[threadIdx.x] = b;
    __syncthreads();
    if (lane == 0 && c < p.C) {
      for (int w = 1; w < 256 / GN_PC; ++w) {
        a += da[w * GN_PC + threadIdx.x];
        b += db[w * GN_PC + threadIdx.x];
      }
      if (p.dbeta) p.dbeta[c] = (float)(a + (p.acc_par ? (double)p.dbeta[c] : 0.0));
      if (p.dgamma) p.dgamma[c] = (float)(b + (p.acc_par ? (double)p.dgamma[c] : 0.0));
    }
    return;
  }
  const int blk = blockIdx.x - npar, n = blk / p.chunks, j = blk % p.chunks;
  const int r0 = j * p.rows, nr = min(p.HW - r0, p.rows);
  {
    const int L = join_lanes(p.G), gl = threadIdx.x % L, gstep = 256 / L;
    const float2* part = p.gpart + (size_t)n * p.chunks * p.G;
    const double inv = 1.0 / ((double)p.HW * p.cg);
    for (int g0 = 0; g0 < p.G; g0 += gstep) {
      const int g = g0 + threadIdx.x / L;
      double a = 0.0, b = 0.0;
      if (g < p.G)
        for (int i = gl; i < p.chunks; i += L) {
          const float2 o = part[(size_t)i * p.G + g];
          a += (double)o.x;
          b += (double)o.y;
        }
      a = lane_sum(a, L);
      b = lane_sum(b, L);
      if (g < p.G && gl == 0) {
        gm[2 * g] = (float)(a * inv);
        gm[2 * g + 1] = (float)(b * inv);
      }
    }
  }
  __syncthreads();
  const int cv = p.C / V, cols = min(cv, 256), rpb = 256 / cols;
  const int tcol = threadIdx.x % cols, trow = threadIdx.x / cols;
  if (trow >= rpb) return;
  const size_t row0 = (size_t)n * p.HW + r0;
  const float* st = p.stats + (size_t)n * 2 * p.G;
  for (int col = tcol; col < cv; col += cols) {
    float mu[V], rs[V], ga[V], be[V], m1[V], m2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = col * V + e, g = c / p.cg;
      mu[e] = st[2 * g];
      rs[e] = st[2 * g + 1];
      ga[e] = p.gamma ? p.gamma[c] : 1.f;
      be[e] = p.beta ? p.beta[c] : 0.f;
      m1[e] = gm[2 * g];
      m2[e] = gm[2 * g + 1];
    }
    const T* px = (const T*)p.x + row0 * p.x_ld + (size_t)col * V;
    const T* pd = (const T*)p.dout + row0 * p.d_ld + (size_t)col * V;
    T* po = (T*)p.out + row0 * p.o_ld + (size_t)col * V;
#pragma unroll 2
    for (int r = trow; r < nr; r += rpb) {
      float f[V], d[V], o[V];
      Lane<T, V>::load(px + (size_t)r * p.x_ld, f);
      Lane<T, V>::load(pd + (size_t)r * p.d_ld, d);
      if (p.acc_dx) Lane<T, V>::load(po + (size_t)r * p.o_ld, o);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xh = (f[e] - mu[e]) * rs[e];
        const float v = ga[e] * d[e] * act_grad<Vec<T>::precise>(fmaf(ga[e], xh, be[e]), act);
        const float g = rs[e] * (v - m1[e] - xh * m2[e]);
        d[e] = p.acc_dx ? o[e] + g : g;
      }
      Lane<T, V>::store(po + (size_t)r * p.o_ld, d);
    }
  }
}

// ------------------------------------------------------------------------------------------------ host side
// Row chunks of one image.  A function of the descriptor's sizes alone, so that the workspace does not depend on addresses: about eight
// workgroups per compute unit over the whole batch, and at least 8192 values per chunk.
void gn_chunks(const plyolo_gn_desc* d, int* chunks, int* rows) {
  const int64_t all = (int64_t)d->N * d->HW;
  int64_t r = (all + 2047) / 2048;
  const int64_t least = (8192 + d->C - 1) / d->C;
  if (r < least) r = least;
  if (r > d->HW) r = d->HW;
  *rows = (int)r;
  *chunks = (int)((d->HW + r - 1) / r);
}

int check_gn(const plyolo_gn_desc* d, const char* who) {
  PLY_CHECK_ARG(d != nullptr, "%s: null descriptor", who);
  PLY_CHECK_ARG(d->dtype == PLYOLO_BF16 || d->dtype == PLYOLO_F32, "%s: bad dtype %d", who, d->dtype);
  PLY_CHECK_ARG(d->N > 0 && d->HW > 0 && d->C > 0 && d->groups > 0, "%s: non-positive dimension (N %d, HW %d, C %d, groups %d)", who, d->N, d->HW, d->C, d->groups);
  PLY_CHECK_ARG(d->C % d->groups == 0, "%s: %d channels do not split into %d groups", who, d->C, d->groups);
  PLY_CHECK_ARG(d->C <= GN_MAXC, "%s: more than %d channels (%d)", who, GN_MAXC, d->C);
  PLY_CHECK_ARG((double)d->N * d->HW < 2147483648.0, "%s: more than 2^31 rows", who);
  PLY_CHECK_ARG(d->act >= PLYOLO_ACT_NONE && d->act <= PLYOLO_ACT_GELU, "%s: bad activation %d", who, d->act);
  PLY_CHECK_ARG(d->eps >= 0.f, "%s: eps must not be negative", who);
  PLY_CHECK_ARG(d->x_ld >= d->C, "%s: x_ld %d < C %d", who, d->x_ld, d->C);
  return 0;
}

size_t gn_ws_bytes(const plyolo_gn_desc* d) {
  int chunks, rows;
  gn_chunks(d, &chunks, &rows);
  return (size_t)d->N * chunks * ((size_t)d->groups + d->C) * sizeof(float2) + (size_t)d->N * d->groups * sizeof(float);
}

GnP gn_params(const plyolo_gn_desc* d, void* ws) {
  GnP p{};
  p.N = d->N; p.HW = d->HW; p.C = d->C; p.G = d->groups; p.cg = d->C / d->groups; p.act = d->act;
  p.x_ld = d->x_ld; p.r_ld = d->r_ld; p.eps = d->eps;
  gn_chunks(d, &p.chunks, &p.rows);
  p.gpart = (float2*)ws;
  p.cpart = p.gpart + (size_t)p.N * p.chunks * p.G;
  p.origin = (float*)(p.cpart + (size_t)p.N * p.chunks * p.C);
  return p;
}

#define GN_DISPATCH(dtype, wide, act, KERN)                                                                                     \
  ((dtype) == PLYOLO_BF16 ? ((wide) ? ((act) == PLYOLO_ACT_SILU ? KERN<bf16_t, 8, PLYOLO_ACT_SILU> : KERN<bf16_t, 8, -1>)         \
                                    : KERN<bf16_t, 1, -1>)                                                                      \
                          : ((wide) ? ((act) == PLYOLO_ACT_SILU ? KERN<float, 4, PLYOLO_ACT_SILU> : KERN<float, 4, -1>) : KERN<float, 1, -1>))

}  // namespace

extern "C" {

size_t plyolo_gn_workspace(const plyolo_gn_desc* d) {
  if (check_gn(d, "gn_workspace")) return 0;
  return gn_ws_bytes(d);
}

int plyolo_gn_act_fwd(const plyolo_gn_desc* d, const void* x, const float* gamma, const float* beta, const void* res, void* out, float* stats,
                      void* workspace, size_t ws_bytes, void* stream) {
  if (check_gn(d, "gn_act_fwd")) return -1;
  PLY_CHECK_ARG(x && out && stats, "gn_act_fwd: null operand");
  PLY_CHECK_ARG(d->o_ld >= d->C && (!res || d->r_ld >= d->C), "gn_act_fwd: o_ld %d or r_ld %d < C %d", d->o_ld, d->r_ld, d->C);
  const size_t es = d->dtype == PLYOLO_BF16 ? 2 : 4;
  PLY_CHECK_ARG(((size_t)x | (size_t)out | (size_t)res) % es == 0 && ((size_t)gamma | (size_t)beta | (size_t)stats) % 4 == 0, "gn_act_fwd: misaligned operand");
  PLY_CHECK_ARG(workspace && (size_t)workspace % 16 == 0 && ws_bytes >= gn_ws_bytes(d), "gn_act_fwd: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", gn_ws_bytes(d), ws_bytes);
  GnP p = gn_params(d, workspace);
  p.x = x; p.res = res; p.out = out; p.gamma = gamma; p.beta = beta; p.stats = stats; p.o_ld = d->o_ld;
  const int V = d->dtype == PLYOLO_BF16 ? 8 : 4, dtype = d->dtype, act = d->act;
  const bool wide = d->C % V == 0 && d->x_ld % V == 0 && d->o_ld % V == 0 && (!res || d->r_ld % V == 0) && ((size_t)x | (size_t)out | (size_t)res) % 16 == 0;
  plyolo::annotate("gn_act_fwd", 0.0, (double)p.N * p.HW * p.C * es * (res ? 3.0 : 2.0));
  return plyolo::submit(stream, [=](hipStream_t s) -> hipError_t {
    const dim3 grid((unsigned)p.N * p.chunks), blk(256);
    auto ks = dtype == PLYOLO_BF16 ? (wide ? gn_stats_kernel<bf16_t, 8> : gn_stats_kernel<bf16_t, 1>) : (wide ? gn_stats_kernel<float, 4> : gn_stats_kernel<float, 1>);
    const size_t lc = (size_t)p.C * sizeof(float2), lg = (size_t)p.G * sizeof(float2);
    if (hipError_t e = plyolo::ensure_dynamic_lds((const void*)ks, lc); e != hipSuccess) return e;
    hipLaunchKernelGGL(ks, grid, blk, lc, s, p);
    auto ka = GN_DISPATCH(dtype, wide, act, gn_apply_kernel);
    if (hipError_t e = plyolo::ensure_dynamic_lds((const void*)ka, lg); e != hipSuccess) return e;
    hipLaunchKernelGGL(ka, grid, blk, lg, s, p);
    return hipGetLastError();
  });
}

int plyolo_gn_act_bwd(const plyolo_gn_desc* d, const void* dout, int d_ld, const void* x, const float* stats, const float* gamma,
                      const float* beta, void* dx, int dx_ld, int accumulate_dx, float* dgamma, float* dbeta, int accumulate_params,
                      void* workspace, size_t ws_bytes, void* stream) {
  if (check_gn(d, "gn_act_bwd")) return -1;
  PLY_CHECK_ARG(dout && x && stats && dx, "gn_act_bwd: null operand");
  PLY_CHECK_ARG(d_ld >= d->C && dx_ld >= d->C, "gn_act_bwd: d_ld %d or dx_ld %d < C %d", d_ld, dx_ld, d->C);
  const size_t es = d->dtype == PLYOLO_BF16 ? 2 : 4;
  PLY_CHECK_ARG(((size_t)x | (size_t)dout | (size_t)dx) % es == 0 && ((size_t)gamma | (size_t)beta | (size_t)stats | (size_t)dgamma | (size_t)dbeta) % 4 == 0,
                "gn_act_bwd: misaligned operand");
  PLY_CHECK_ARG(workspace && (size_t)workspace % 16 == 0 && ws_bytes >= gn_ws_bytes(d), "gn_act_bwd: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", gn_ws_bytes(d), ws_bytes);
  GnP p = gn_params(d, workspace);
  p.x = x; p.dout = dout; p.out = dx; p.gamma = gamma; p.beta = beta; p.stats = (float*)stats;
  p.dgamma = dgamma; p.dbeta = dbeta; p.d_ld = d_ld; p.o_ld = dx_ld; p.acc_dx = accumulate_dx ? 1 : 0; p.acc_par = accumulate_params ? 1 : 0;
  const int V = d->dtype == PLYOLO_BF16 ? 8 : 4, dtype = d->dtype, act = d->act;
  const bool wide = d->C % V == 0 && d->x_ld % V == 0 && d_ld % V == 0 && dx_ld % V == 0 && ((size_t)x | (size_t)dout | (size_t)dx) % 16 == 0;
  plyolo::annotate("gn_act_bwd", 0.0, (double)p.N * p.HW * p.C * es * (accumulate_dx ? 4.0 : 3.0));
  return plyolo::submit(stream, [=](hipStream_t s) -> hipError_t {
    const unsigned nblk = (unsigned)p.N * p.chunks;
    const int npar = (p.dgamma || p.dbeta) ? (p.C + GN_PC - 1) / GN_PC : 0;
    const dim3 blk(256);
    const size_t lc = (size_t)p.C * sizeof(float2), lg = (size_t)p.G * sizeof(float2);
    auto ks = GN_DISPATCH(dtype, wide, act, gn_bwd_sums_kernel);
    if (hipError_t e = plyolo::ensure_dynamic_lds((const void*)ks, lc); e != hipSuccess) return e;
    hipLaunchKernelGGL(ks, dim3(nblk), blk, lc, s, p);
    auto kd = GN_DISPATCH(dtype, wide, act, gn_bwd_dx_kernel);
    if (hipError_t e = plyolo::ensure_dynamic_lds((const void*)kd, lg); e != hipSuccess) return e;
    hipLaunchKernelGGL(kd, dim3(nblk + npar), blk, lg, s, p, npar);
    return hipGetLastError();
  });
}

}  // extern "C"
