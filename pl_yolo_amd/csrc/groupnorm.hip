// Group norm + activation (+ shortcut) on channels-last rows, forward and backward.
//
//   xh = (x - mean) rstd,  u = gamma xh + beta,  out = act(u) + res          mean, rstd over the HW * C/groups values of (image, group)
//   du = dout act'(u),  dbeta = sum du,  dgamma = sum du xh,  v = gamma du
//   dx = rstd (v - mean(v) - xh mean(v xh))                                  means over the same (image, group)
//
// Both directions are HBM streams around one reduction.
//   resident   a workgroup owns (image, slice of whole groups) and holds its rows in registers across the reduction: one launch, every
//              operand read once (gn_res_*_kernel).  Taken wherever the slice fits.
//   streaming  three launches: partials per (image, chunk of rows) into the workspace, a join of the partials in a fixed order, the stream.
//              (Joining in the stream's own prologue saves a launch and loses more: every workgroup then reads all partials of its image, and
//              all of them the same lines at the same time -- 1 x 25600 x 64 forward 35 us at 400 chunks, 87 us at 800.)
// A thread owns one vector of channels for the whole launch and walks down the rows, as in the BatchNorm kernels.
//
// The variance is never formed as E[x^2] - E[x]^2: a thread sums deviations from its own first value, (count, mean, M2) triples are joined
// by Chan's formula, and the means of the triples are kept as distances from the first value of their (image, group): neither a mean of
// thousands of spreads nor one huge value costs digits.
//
// Times in this file are of whole calls in a captured graph that goes over three sets of operands in turn (more than the last-level cache
// holds comes from HBM); "cached": over one set.  Times of single kernels are the profiler's, over three sets as well.
#include "common.h"

namespace {

constexpr int GN_MAXC = 4096;    // channels (LDS: two floats each)

typedef u32x4 __attribute__((aligned(2))) u32x4_any;     // 16 bytes at any element address: the same instruction as the aligned access
typedef f32x4 __attribute__((aligned(4))) f32x4_any;

// V channels of one row: a 16-byte vector (8 bf16, 4 fp32) at any element address, or (V == 1) one element
template <typename T, int V> struct Lane;
template <> struct Lane<bf16_t, 8> {
  typedef u32x4 raw;
  static DEVINL raw get(const bf16_t* p) { return *(const u32x4_any*)p; }
  static DEVINL void cvt(const raw& v, float (&f)[8]) { Vec<bf16_t>::cvt(v, f); }
  static DEVINL void store(bf16_t* p, const float (&f)[8]) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pack2bf(f[2 * i], f[2 * i + 1]);
    *(u32x4_any*)p = v;
  }
};
template <> struct Lane<float, 4> {
  typedef f32x4 raw;
  static DEVINL raw get(const float* p) { return *(const f32x4_any*)p; }
  static DEVINL void cvt(const raw& v, float (&f)[4]) { Vec<float>::cvt(v, f); }
  static DEVINL void store(float* p, const float (&f)[4]) { *(f32x4_any*)p = f32x4{f[0], f[1], f[2], f[3]}; }
};
template <typename T> struct Lane<T, 1> {
  typedef T raw;
  static DEVINL raw get(const T* p) { return *p; }
  static DEVINL void cvt(const raw& v, float (&f)[1]) { f[0] = ActT<T>::ld(&v); }
  static DEVINL void store(T* p, const float (&f)[1]) { ActT<T>::st(p, f[0]); }
};
template <typename T, int V> DEVINL void lane_load(const T* p, float (&f)[V]) { Lane<T, V>::cvt(Lane<T, V>::get(p), f); }

// act(u) and act'(u).  bf16 SiLU is written out: both passes of the backward recompute it, and at 8 TB/s the vector ALU has about fifteen
// issue slots per element (the hardware exponential and reciprocal take four each)
template <bool PRECISE> DEVINL float gn_act(float u, int act) { return actf<PRECISE>(u, act); }
template <bool PRECISE> DEVINL float gn_act_grad(float u, int act) {
  if (!PRECISE && act == PLYOLO_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(u * -1.4426950408889634f));
    return fmaf(s, fmaf(-u, s, u), s);
  }
  return act_grad<PRECISE>(u, act);
}

struct GnP {
  const void* x;
  const void* dout;
  const void* res;
  void* out;           // forward: out; backward: dx
  const float* gamma;
  const float* beta;
  float* stats;        // [N][G][2]
  float2* gpart;       // [N][chunks][G]: forward (mean - origin, M2), backward (sum v, sum v xh)
  float2* gmean;       // [N][G]: backward (mean v, mean v xh)
  float2* cpart;       // [N][chunks][C]: backward (sum du, sum du xh)
  float* dgamma;
  float* dbeta;
  int N, HW, C, G, cg, act;
  int x_ld, d_ld, r_ld, o_ld;
  int chunks, rows;    // row chunks per image, rows per chunk
  int acc_dx, acc_par;
  float eps, inv_cg;   // 1 / cg
  double inv_count;    // 1 / (HW cg)
};
// c / cg without an integer division: c + 1/2 is at least 1 / (2 cg) from every multiple of cg, relative 2^-13 at c <= 4096, and the product is
// off by 2^-23
DEVINL int group_of(const GnP& p, int c) { return (int)(((float)c + 0.5f) * p.inv_cg); }

// 2^lane_shift lanes share the reduction of one of n items: as many as nt threads have for it, a wave at most
DEVINL int lane_shift(int n, int nt) {
  int s = 6;
  while (s > 0 && (n << s) > nt) --s;
  return s;
}
template <typename A> DEVINL A lane_sum(A v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// ------------------------------------------------------------------------------------------------ forward
// Vector `col` of a row of any C >= V channels (streaming kernels): the last one of a row that V does not divide is the row's last V channels,
// of which the first `skip` are its neighbour's -- read, never summed or stored.  (Element by element instead: 16 x 6400 x 132 bf16 forward 44,
// backward 138 us; this way 33 and 46.)
// RAG: there is such a vector (8 x 25600 x 320 backward 149 us with the test for it, 146 without; cached 127 and 124).
template <int V, bool RAG> struct Col {
  int c, skip;
  DEVINL Col(const GnP& p, int col) : c(RAG ? min(col * V, p.C - V) : col * V), skip(RAG ? col * V - c : 0) {}
};
template <typename T, int V> DEVINL void store_from(T* p, const float (&f)[V], int skip) {
  if (skip == 0) {
    Lane<T, V>::store(p, f);
    return;
  }
#pragma unroll
  for (int e = 1; e < V; ++e)
    if (e >= skip) ActT<T>::st(p + e, f[e]);
}

// the value from which the means of (image, group) are counted
template <typename T> DEVINL float gn_origin(const GnP& p, int n, int g) {
  return ActT<T>::ld((const T*)p.x + (size_t)n * p.HW * p.x_ld + (size_t)g * p.cg);
}

// (mean - origin, M2) of every group over the rows of one chunk: one read of x, a thread's deviations are taken from its own first value
template <typename T, int V, bool RAG> __global__ __launch_bounds__(256) void gn_stats_kernel(const GnP p) {
  extern __shared__ float2 chan[];             // [C] (mean - origin, M2) of one channel over the chunk
  __shared__ float2 red[256 * V];
  const int n = blockIdx.x / p.chunks, j = blockIdx.x % p.chunks;
  const int r0 = j * p.rows, nr = min(p.HW - r0, p.rows);
  const int cv = (p.C + V - 1) / V, cols = min(cv, 256), rpb = 256 / cols;
  const int tcol = threadIdx.x % cols, trow = threadIdx.x / cols;
  const T* base = (const T*)p.x + ((size_t)n * p.HW + r0) * p.x_ld;
  for (int cb = 0; cb < cv; cb += cols) {
    const int col = cb + tcol;
    if (col < cv && trow < rpb) {
      const Col<V, RAG> at(p, col);
      const T* px = base + at.c;
      float k[V], s[V], q[V], f[V];
#pragma unroll
      for (int e = 0; e < V; ++e) k[e] = s[e] = q[e] = 0.f;
      if (trow < nr) lane_load<T, V>(px + (size_t)trow * p.x_ld, k);
      int cnt = trow < nr ? 1 : 0;
#pragma unroll 4
      for (int r = trow + rpb; r < nr; r += rpb) {
        lane_load<T, V>(px + (size_t)r * p.x_ld, f);
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
        const float from = k[e] - gn_origin<T>(p, n, group_of(p, at.c + e));
        if (e >= at.skip) red[(trow * cols + tcol) * V + e - at.skip] = make_float2(from + s[e] * inv, m2 < 0.f ? 0.f : m2);   // (a NaN passes)
      }
    }
    __syncthreads();
    const int nch = min(cols * V, p.C - cb * V), nrow = min(rpb, nr), per = nr / rpb, extra = nr % rpb;
    const int sh = lane_shift(nch, 256), L = 1 << sh, lane = threadIdx.x & (L - 1);
    for (int k = 0; k < nch; k += 256 >> sh) {
      const int t = k + (threadIdx.x >> sh);
      const bool live = t < nch;
      float mean = 0.f, m2 = 0.f;
      if (live)
        for (int w = lane; w < nrow; w += L) mean = fmaf(red[w * cols * V + t].x, (float)(per + (w < extra ? 1 : 0)), mean);
      mean = lane_sum(mean, L) / (float)nr;
      if (live)
        for (int w = lane; w < nrow; w += L) {
          const float2 o = red[w * cols * V + t];
          const float d = o.x - mean;
          m2 += fmaf(d * d, (float)(per + (w < extra ? 1 : 0)), o.y);
        }
      m2 = lane_sum(m2, L);
      if (live && lane == 0) chan[cb * V + t] = make_float2(mean, m2);
    }
    __syncthreads();
  }
  // channels -> groups: equal counts, so the group's mean is the mean of means
  const int sh = lane_shift(p.G, 256), L = 1 << sh, gl = threadIdx.x & (L - 1), gstep = 256 >> sh;
  for (int g0 = 0; g0 < p.G; g0 += gstep) {
    const int g = g0 + (threadIdx.x >> sh);
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
    if (on && gl == 0) p.gpart[((size_t)n * p.chunks + j) * p.G + g] = make_float2(mean, m2);
  }
}

// Joins: 32 items (groups of an image, or channels) x NT / 32 lanes per workgroup, a lane's partials requested sixteen at a time, lanes added
// in a fixed order.  fp64: the two sums of a group are then enough, however far its mean lies from the origin.
constexpr int JOIN_I = 32, JOIN_FEW = 128;      // up to that many partials eight lanes per item do (NT 256; beyond, 32 lanes)
template <int JOIN_NT> DEVINL void join_sums(const float2* part, int stride, int count, bool live, double& a, double& b, const double full, const double tail) {
  __shared__ double da[JOIN_NT], db[JOIN_NT];
  const int lane = threadIdx.x / JOIN_I, last = count - 1;
  a = b = 0.0;
  if (live)
    for (int j0 = lane; j0 < count; j0 += 16 * (JOIN_NT / JOIN_I)) {
      float2 o[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) o[k] = part[(size_t)min(j0 + k * (JOIN_NT / JOIN_I), last) * stride];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int j = j0 + k * (JOIN_NT / JOIN_I);
        if (j > last) continue;
        if (full > 0.0) {      // (mean - origin, M2) of `full` values (the last: `tail`; more than a float counts) -> sum, sum of squares
          const double w = j < last ? full : tail;
          a += w * (double)o[k].x;
          b += (double)o[k].y + w * (double)o[k].x * (double)o[k].x;
        } else {
          a += (double)o[k].x;
          b += (double)o[k].y;
        }
      }
    }
  da[threadIdx.x] = a;
  db[threadIdx.x] = b;
  __syncthreads();
  for (int h = JOIN_NT / 2; h >= JOIN_I; h >>= 1) {
    if ((int)threadIdx.x < h) {
      da[threadIdx.x] += da[threadIdx.x + h];
      db[threadIdx.x] += db[threadIdx.x + h];
    }
    __syncthreads();
  }
  a = da[threadIdx.x % JOIN_I];
  b = db[threadIdx.x % JOIN_I];
}

template <typename T, int JOIN_NT> __global__ __launch_bounds__(JOIN_NT) void gn_join_fwd_kernel(const GnP p) {
  const int gb = (p.G + JOIN_I - 1) / JOIN_I, n = blockIdx.x / gb, g = (blockIdx.x % gb) * JOIN_I + threadIdx.x % JOIN_I;
  const bool live = g < p.G;
  double s, q;
  join_sums<JOIN_NT>(p.gpart + (size_t)n * p.chunks * p.G + g, p.G, p.chunks, live, s, q, (double)p.rows * p.cg,
            (double)(p.HW - (p.chunks - 1) * p.rows) * p.cg);
  if (live && (int)threadIdx.x < JOIN_I) {
    const double total = (double)p.HW * p.cg, mean = s / total, m2 = q - s * mean;
    float* st = p.stats + ((size_t)n * p.G + g) * 2;
    st[0] = (float)(mean + (double)gn_origin<T>(p, n, g));
    st[1] = (float)rsqrt((m2 < 0.0 ? 0.0 : m2) * p.inv_count + (double)p.eps);
  }
}

constexpr int GN_U = 4;    // rows a thread has in flight

// the stream of the forward: GN_U rows requested ahead of the GN_U being formed (statistics, join and this: 32 x 6400 x 256 bf16 75 us, 2.8 TB/s
// counting x once)
template <typename T, int V, int ACTC, bool RAG> __global__ __launch_bounds__(256) void gn_apply_kernel(const GnP p) {
  // last chunk first: what the statistics read last is still in the last-level cache
  const int blk = gridDim.x - 1 - blockIdx.x, n = blk / p.chunks, j = blk % p.chunks;
  const int r0 = j * p.rows, nr = min(p.HW - r0, p.rows);
  const int act = ACTC >= 0 ? ACTC : p.act;
  const int cv = (p.C + V - 1) / V, cols = min(cv, 256), rpb = 256 / cols;
  const int tcol = threadIdx.x % cols, trow = threadIdx.x / cols;
  const size_t row0 = (size_t)n * p.HW + r0;
  typedef typename Lane<T, V>::raw raw_t;
  raw_t rx[GN_U], rr[GN_U];
  const bool rows_mine = trow < rpb;
  auto request = [&](const int col, const int r) {
    const Col<V, RAG> at(p, col);
    const T* px = (const T*)p.x + row0 * p.x_ld + at.c;
    const T* pr = (const T*)p.res + row0 * p.r_ld + at.c;
#pragma unroll
    for (int u = 0; u < GN_U; ++u)
      if (r + u * rpb < nr) {
        rx[u] = Lane<T, V>::get(px + (size_t)(r + u * rpb) * p.x_ld);
        if (p.res) rr[u] = Lane<T, V>::get(pr + (size_t)(r + u * rpb) * p.r_ld);
      }
  };
  float a[V], b[V], mu[V];
  if (!rows_mine) return;
  const float* st = p.stats + (size_t)n * 2 * p.G;
  for (int col = tcol; col < cv; col += cols) {
    const Col<V, RAG> at(p, col);
    request(col, trow);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = at.c + e, g = group_of(p, c);
      mu[e] = st[2 * g];
      a[e] = st[2 * g + 1] * (p.gamma ? p.gamma[c] : 1.f);
      b[e] = p.beta ? p.beta[c] : 0.f;
    }
    T* po = (T*)p.out + row0 * p.o_ld + at.c;
    for (int r = trow; r < nr; r += GN_U * rpb) {
      raw_t cx[GN_U], cr[GN_U];
#pragma unroll
      for (int u = 0; u < GN_U; ++u) {
        cx[u] = rx[u];
        cr[u] = rr[u];
      }
      request(col, r + GN_U * rpb);
#pragma unroll
      for (int u = 0; u < GN_U; ++u)
        if (r + u * rpb < nr) {
          float f[V], t[V];
          Lane<T, V>::cvt(cx[u], f);
          if (p.res) Lane<T, V>::cvt(cr[u], t);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            f[e] = gn_act<Vec<T>::precise>(fmaf(f[e] - mu[e], a[e], b[e]), act);
            if (p.res) f[e] += t[e];
          }
          store_from<T, V>(po + (size_t)(r + u * rpb) * p.o_ld, f, at.skip);
        }
    }
  }
}

// ------------------------------------------------------------------------------------------------ backward
constexpr int GN_BU = 2;   // rows of x and dout a thread has in flight

template <typename T, int V>
DEVINL void gn_request(typename Lane<T, V>::raw (&rx)[GN_BU], typename Lane<T, V>::raw (&rd)[GN_BU], const T* px, const T* pd, const GnP& p, int r, int nr, int rpb) {
#pragma unroll
  for (int u = 0; u < GN_BU; ++u)
    if (r + u * rpb < nr) {
      rx[u] = Lane<T, V>::get(px + (size_t)(r + u * rpb) * p.x_ld);
      rd[u] = Lane<T, V>::get(pd + (size_t)(r + u * rpb) * p.d_ld);
    }
}

// per chunk: (sum du, sum du xh) of every channel, and (sum v, sum v xh) of every group.  Reads: 8 x 25600 x 320 bf16 74 us, 3.5 TB/s
// from HBM (cached 54 us); every byte of x and dout is fetched once
template <typename T, int V, int ACTC, bool RAG> __global__ __launch_bounds__(256) void gn_bwd_sums_kernel(const GnP p) {
  extern __shared__ float2 chan[];
  __shared__ float2 red[256 * V];
  const int n = blockIdx.x / p.chunks, j = blockIdx.x % p.chunks;
  const int r0 = j * p.rows, nr = min(p.HW - r0, p.rows);
  const int act = ACTC >= 0 ? ACTC : p.act;
  const int cv = (p.C + V - 1) / V, cols = min(cv, 256), rpb = 256 / cols;
  const int tcol = threadIdx.x % cols, trow = threadIdx.x / cols;
  const size_t row0 = (size_t)n * p.HW + r0;
  const float* st = p.stats + (size_t)n * 2 * p.G;
  float2* cp = p.cpart + ((size_t)n * p.chunks + j) * p.C;
  for (int cb = 0; cb < cv; cb += cols) {
    const int col = cb + tcol;
    if (col < cv && trow < rpb) {
      const Col<V, RAG> at(p, col);
      float mu[V], rs[V], ga[V], be[V], sa[V], sb[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int c = at.c + e, g = group_of(p, c);
        mu[e] = st[2 * g];
        rs[e] = st[2 * g + 1];
        ga[e] = rs[e] * (p.gamma ? p.gamma[c] : 1.f);
        be[e] = p.beta ? p.beta[c] : 0.f;
        sa[e] = sb[e] = 0.f;
      }
      const T* px = (const T*)p.x + row0 * p.x_ld + at.c;
      const T* pd = (const T*)p.dout + row0 * p.d_ld + at.c;
      typename Lane<T, V>::raw rx[GN_BU], rd[GN_BU], cx[GN_BU], cd[GN_BU];
      gn_request<T, V>(rx, rd, px, pd, p, trow, nr, rpb);
      for (int r = trow; r < nr; r += GN_BU * rpb) {
#pragma unroll
        for (int u = 0; u < GN_BU; ++u) {
          cx[u] = rx[u];
          cd[u] = rd[u];
        }
        gn_request<T, V>(rx, rd, px, pd, p, r + GN_BU * rpb, nr, rpb);
#pragma unroll
        for (int u = 0; u < GN_BU; ++u)
          if (r + u * rpb < nr) {
            float f[V], d[V];
            Lane<T, V>::cvt(cx[u], f);
            Lane<T, V>::cvt(cd[u], d);
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float c = f[e] - mu[e];                     // xh = rs c
              const float du = d[e] * gn_act_grad<Vec<T>::precise>(fmaf(ga[e], c, be[e]), act);
              sa[e] += du;
              sb[e] = fmaf(du, c, sb[e]);
            }
          }
      }
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e >= at.skip) red[(trow * cols + tcol) * V + e - at.skip] = make_float2(sa[e], sb[e] * rs[e]);
    }
    __syncthreads();
    const int nch = min(cols * V, p.C - cb * V), nrow = min(rpb, nr);
    const int sh = lane_shift(nch, 256), L = 1 << sh, lane = threadIdx.x & (L - 1);
    for (int k = 0; k < nch; k += 256 >> sh) {
      const int t = k + (threadIdx.x >> sh), c = cb * V + t;
      const bool live = t < nch;
      float a = 0.f, b = 0.f;
      if (live)
        for (int w = lane; w < nrow; w += L) {
          const float2 o = red[w * cols * V + t];
          a += o.x;
          b += o.y;
        }
      a = lane_sum(a, L);
      b = lane_sum(b, L);
      if (live && lane == 0) {
        chan[c] = make_float2(a, b);
        cp[c] = make_float2(a, b);
      }
    }
    __syncthreads();
  }
  const int sh = lane_shift(p.G, 256), L = 1 << sh, gl = threadIdx.x & (L - 1), gstep = 256 >> sh;
  for (int g0 = 0; g0 < p.G; g0 += gstep) {
    const int g = g0 + (threadIdx.x >> sh);
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

// workgroups [0, npar): dgamma / dbeta of 32 channels from `parts` per-channel partials; the others: the two means of 32 groups of an image
template <int JOIN_NT> __global__ __launch_bounds__(JOIN_NT) void gn_join_bwd_kernel(const GnP p, const int npar, const int parts) {
  double a, b;
  if ((int)blockIdx.x < npar) {
    const int c = blockIdx.x * JOIN_I + threadIdx.x % JOIN_I;
    join_sums<JOIN_NT>(p.cpart + c, p.C, parts, c < p.C, a, b, 0.0, 0.0);
    if (c < p.C && (int)threadIdx.x < JOIN_I) {
      if (p.dbeta) p.dbeta[c] = (float)(a + (p.acc_par ? (double)p.dbeta[c] : 0.0));
      if (p.dgamma) p.dgamma[c] = (float)(b + (p.acc_par ? (double)p.dgamma[c] : 0.0));
    }
    return;
  }
  const int blk = blockIdx.x - npar, gb = (p.G + JOIN_I - 1) / JOIN_I, n = blk / gb, g = (blk % gb) * JOIN_I + threadIdx.x % JOIN_I;
  join_sums<JOIN_NT>(p.gpart + (size_t)n * p.chunks * p.G + g, p.G, p.chunks, g < p.G, a, b, 0.0, 0.0);
  if (g < p.G && (int)threadIdx.x < JOIN_I) {
    const double inv = p.inv_count;
    p.gmean[(size_t)n * p.G + g] = make_float2((float)(a * inv), (float)(b * inv));
  }
}

// the stream of the backward.  HBM: 8 x 25600 x 320 bf16 67 us, 5.9 TB/s (part of what the sums read last is still in the last-level cache)
template <typename T, int V, int ACTC, bool RAG> __global__ __launch_bounds__(256) void gn_bwd_dx_kernel(const GnP p) {
  const int act = ACTC >= 0 ? ACTC : p.act;
  const int blk = gridDim.x - 1 - blockIdx.x, n = blk / p.chunks, j = blk % p.chunks;      // last chunk first, as in gn_apply_kernel
  const int r0 = j * p.rows, nr = min(p.HW - r0, p.rows);
  const int cv = (p.C + V - 1) / V, cols = min(cv, 256), rpb = 256 / cols;
  const int tcol = threadIdx.x % cols, trow = threadIdx.x / cols;
  if (trow >= rpb) return;
  const size_t row0 = (size_t)n * p.HW + r0;
  const float* st = p.stats + (size_t)n * 2 * p.G;
  const float2* gm = p.gmean + (size_t)n * p.G;
  for (int col = tcol; col < cv; col += cols) {
    const Col<V, RAG> at(p, col);
    float mu[V], ga[V], be[V], k0[V], k1[V];      // dx = (rs gamma) du + k0 + k1 c with c = x - mean
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = at.c + e, g = group_of(p, c);
      const float rs = st[2 * g + 1];
      mu[e] = st[2 * g];
      ga[e] = rs * (p.gamma ? p.gamma[c] : 1.f);
      be[e] = p.beta ? p.beta[c] : 0.f;
      k0[e] = -rs * gm[g].x;
      k1[e] = -rs * rs * gm[g].y;
    }
    const T* px = (const T*)p.x + row0 * p.x_ld + at.c;
    const T* pd = (const T*)p.dout + row0 * p.d_ld + at.c;
    T* po = (T*)p.out + row0 * p.o_ld + at.c;
    typename Lane<T, V>::raw rx[GN_BU], rd[GN_BU], cx[GN_BU], cd[GN_BU];
    gn_request<T, V>(rx, rd, px, pd, p, trow, nr, rpb);
    for (int r = trow; r < nr; r += GN_BU * rpb) {
#pragma unroll
      for (int u = 0; u < GN_BU; ++u) {
        cx[u] = rx[u];
        cd[u] = rd[u];
      }
      gn_request<T, V>(rx, rd, px, pd, p, r + GN_BU * rpb, nr, rpb);
#pragma unroll
      for (int u = 0; u < GN_BU; ++u)
        if (r + u * rpb < nr) {
          float f[V], d[V], o[V];
          Lane<T, V>::cvt(cx[u], f);
          Lane<T, V>::cvt(cd[u], d);
          if (p.acc_dx) lane_load<T, V>(po + (size_t)(r + u * rpb) * p.o_ld, o);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float c = f[e] - mu[e];
            const float du = d[e] * gn_act_grad<Vec<T>::precise>(fmaf(ga[e], c, be[e]), act);
            const float g = fmaf(ga[e], du, fmaf(k1[e], c, k0[e]));
            d[e] = p.acc_dx ? o[e] + g : g;
          }
          store_from<T, V>(po + (size_t)(r + u * rpb) * p.o_ld, d, at.skip);
        }
    }
  }
}

// ------------------------------------------------------------------------------------------------ resident slices
// One workgroup = (image, slice of sv vectors that hold whole groups); thread t owns vector column t % sv and rows t / sv + i * rpb, i < NV, as
// raw vectors in registers.  Slices of one image share 128-byte lines, so they get neighbouring ids on one XCD (its L2 serves the line's
// other readers).
constexpr int RES_NT = 512;

struct ResP {
  GnP g;
  int sv, slices, rpb;     // vectors per slice, slices per image, rows per pass of the workgroup
};

DEVINL int xcd_contiguous(int id, int n) {      // hardware deals workgroup ids round robin over the 8 XCDs: give each a contiguous range
  const int q = n >> 3, r = n & 7, x = id & 7;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (id >> 3);
}

// The chip reads, reduces and writes one after the other: 32 x 6400 x 128 bf16 38 us for 105 MB, cached 29;
// on one 400 x 256 image it is a chain of latencies, 6.4 us.
template <typename T, int V, int NV, int ACTC, int NT> __global__ __launch_bounds__(NT) void gn_res_fwd_kernel(const ResP q) {
  const GnP& p = q.g;
  extern __shared__ float2 red[];              // [channel of the vector][thread]: (mean, M2) of the thread's values
  float2* chan = red + V * NT;                 // [channels of the slice] (mean - origin, M2), behind them [groups][2] mean, rstd
  float* gm = (float*)(chan + q.sv * V);
  const int id = xcd_contiguous(blockIdx.x, gridDim.x), n = id / q.slices, c0 = (id % q.slices) * q.sv * V;
  const int tid = threadIdx.x, col = tid % q.sv, row = tid / q.sv, act = ACTC >= 0 ? ACTC : p.act;
  const bool on = row < q.rpb;
  const T* px = (const T*)p.x + (size_t)n * p.HW * p.x_ld + c0 + (size_t)col * V;
  typename Lane<T, V>::raw raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int r = row + i * q.rpb;
    if (on && r < p.HW) raw[i] = Lane<T, V>::get(px + (size_t)r * p.x_ld);
  }
  float o[V], ga[V], be[V];       // what else comes from memory is requested before anything waits
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = c0 + col * V + e;
    o[e] = gn_origin<T>(p, n, group_of(p, c));
    ga[e] = p.gamma ? p.gamma[c] : 1.f;
    be[e] = p.beta ? p.beta[c] : 0.f;
  }
  const T* pr = p.res ? (const T*)p.res + ((size_t)n * p.HW + row) * p.r_ld + c0 + (size_t)col * V : nullptr;
  constexpr int NR = NV <= 4 ? NV : 1;     // (few rows: the shortcut's as well)
  typename Lane<T, V>::raw rres[NR];
  if (NV <= 4 && pr)
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int r = row + i * q.rpb;
      if (on && r < p.HW) rres[i] = Lane<T, V>::get(pr + (size_t)i * q.rpb * p.r_ld);
    }
  const int per = p.HW / q.rpb, extra = p.HW % q.rpb;      // rows of a row lane: per, one more in the first `extra` lanes
  const int cnt = on ? per + (row < extra ? 1 : 0) : 0;
  {
    float s[V], k[V], m2[V], f[V];
    if (cnt > 0) Lane<T, V>::cvt(raw[0], k);
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = m2[e] = 0.f;
#pragma unroll
    for (int i = 1; i < NV; ++i)
      if (i < cnt) {
        Lane<T, V>::cvt(raw[i], f);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = f[e] - k[e];
          s[e] += d;
          m2[e] = fmaf(d, d, m2[e]);
        }
      }
    const float inv = cnt > 0 ? 1.0f / (float)cnt : 0.f;
    if (cnt > 0) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float v = m2[e] - s[e] * s[e] * inv;
        red[e * NT + tid] = make_float2((k[e] - o[e]) + s[e] * inv, v < 0.f ? 0.f : v);
      }
    }
  }
  __syncthreads();
  // row lanes -> channels (a channel's partials are 2^lane_shift(nch, NT) lanes' work, about V each) -> groups
  const int nch = q.sv * V, nrow = min(q.rpb, p.HW);
  {
    const int sh = lane_shift(nch, NT), L = 1 << sh, lane = tid & (L - 1);
    for (int k = 0; k < nch; k += NT >> sh) {
      const int c = k + (tid >> sh);
      const bool live = c < nch;
      const float2* e = red + (live ? (c % V) * NT + c / V : 0);
      float mean = 0.f, m2 = 0.f;
      if (live)
        for (int r = lane; r < nrow; r += L) mean = fmaf(e[r * q.sv].x, (float)(per + (r < extra ? 1 : 0)), mean);
      mean = lane_sum(mean, L) / (float)p.HW;
      if (live)
        for (int r = lane; r < nrow; r += L) {
          const float2 o = e[r * q.sv];
          const float d = o.x - mean;
          m2 += fmaf(d * d, (float)(per + (r < extra ? 1 : 0)), o.y);
        }
      m2 = lane_sum(m2, L);
      if (live && lane == 0) chan[c] = make_float2(mean, m2);
    }
  }
  __syncthreads();
  const int gs = nch / p.cg;
  {
    const int sh = lane_shift(gs, NT), L = 1 << sh, lane = tid & (L - 1);
    for (int k = 0; k < gs; k += NT >> sh) {
      const int g = k + (tid >> sh);
      const bool live = g < gs;
      float mean = 0.f, m2 = 0.f;
      if (live)
        for (int c = g * p.cg + lane; c < (g + 1) * p.cg; c += L) mean += chan[c].x;
      mean = lane_sum(mean, L) / (float)p.cg;
      if (live)
        for (int c = g * p.cg + lane; c < (g + 1) * p.cg; c += L) {
          const float d = chan[c].x - mean;
          m2 += fmaf(d * d, (float)p.HW, chan[c].y);
        }
      m2 = lane_sum(m2, L);
      if (live && lane == 0) {
        const int gg = c0 / p.cg + g;
        const float mu = (float)((double)mean + (double)gn_origin<T>(p, n, gg));
        const float rs = (float)rsqrt((double)m2 * p.inv_count + (double)p.eps);
        gm[2 * g] = mu;
        gm[2 * g + 1] = rs;
        p.stats[((size_t)n * p.G + gg) * 2] = mu;
        p.stats[((size_t)n * p.G + gg) * 2 + 1] = rs;
      }
    }
  }
  __syncthreads();
  if (cnt == 0) return;
  float mu[V], a[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int g = group_of(p, col * V + e);
    mu[e] = gm[2 * g];
    a[e] = gm[2 * g + 1] * ga[e];
  }
  const size_t row0 = (size_t)n * p.HW + row;
  T* po = (T*)p.out + row0 * p.o_ld + c0 + (size_t)col * V;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i < cnt) {
      float f[V], t[V];
      Lane<T, V>::cvt(raw[i], f);
      if (NV <= 4 && pr) Lane<T, V>::cvt(rres[i < NR ? i : 0], t);
      else if (pr) lane_load<T, V>(pr + (size_t)i * q.rpb * p.r_ld, t);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[e] = gn_act<Vec<T>::precise>(fmaf(f[e] - mu[e], a[e], be[e]), act);
        if (pr) f[e] += t[e];
      }
      Lane<T, V>::store(po + (size_t)i * q.rpb * p.o_ld, f);
    }
}

// x and dout held across the reduction: 32 x 1600 x 256 bf16 29 us for 79 MB
template <typename T, int V, int NV, int ACTC> __global__ __launch_bounds__(RES_NT) void gn_res_bwd_kernel(const ResP q) {
  const GnP& p = q.g;
  __shared__ float2 red[V * RES_NT];           // (sum du, sum du c) of the thread's rows, then [channel] totals
  extern __shared__ float2 chan[];             // [channels of the slice] (sum du, sum du xh), behind them [groups][2] means
  const int id = xcd_contiguous(blockIdx.x, gridDim.x), n = id / q.slices, nch = q.sv * V, c0 = (id % q.slices) * nch;
  float2* gmean = chan + nch;
  const int tid = threadIdx.x, col = tid % q.sv, row = tid / q.sv, act = ACTC >= 0 ? ACTC : p.act;
  const int cnt = row < q.rpb ? p.HW / q.rpb + (row < p.HW % q.rpb ? 1 : 0) : 0;
  const size_t row0 = (size_t)n * p.HW + row;
  const T* px = (const T*)p.x + row0 * p.x_ld + c0 + (size_t)col * V;
  const T* pd = (const T*)p.dout + row0 * p.d_ld + c0 + (size_t)col * V;
  typename Lane<T, V>::raw rx[NV], rd[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i < cnt) {
      rx[i] = Lane<T, V>::get(px + (size_t)i * q.rpb * p.x_ld);
      rd[i] = Lane<T, V>::get(pd + (size_t)i * q.rpb * p.d_ld);
    }
  const float* st = p.stats + ((size_t)n * p.G + c0 / p.cg) * 2;
  float mu[V], ga[V], be[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = c0 + col * V + e, g = group_of(p, col * V + e);
    mu[e] = st[2 * g];
    ga[e] = st[2 * g + 1] * (p.gamma ? p.gamma[c] : 1.f);
    be[e] = p.beta ? p.beta[c] : 0.f;
  }
  {
    float sa[V], sb[V], f[V], d[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sa[e] = sb[e] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i < cnt) {
        Lane<T, V>::cvt(rx[i], f);
        Lane<T, V>::cvt(rd[i], d);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float c = f[e] - mu[e];
          const float du = d[e] * gn_act_grad<Vec<T>::precise>(fmaf(ga[e], c, be[e]), act);
          sa[e] += du;
          sb[e] = fmaf(du, c, sb[e]);
        }
      }
    if (cnt > 0) {
#pragma unroll
      for (int e = 0; e < V; ++e) red[e * RES_NT + tid] = make_float2(sa[e], sb[e]);
    }
  }
  __syncthreads();
  const int nrow = min(q.rpb, p.HW);
  {
    const int sh = lane_shift(nch, RES_NT), L = 1 << sh, lane = tid & (L - 1);
    for (int k = 0; k < nch; k += RES_NT >> sh) {
      const int c = k + (tid >> sh);
      const bool live = c < nch;
      const float2* e = red + (live ? (c % V) * RES_NT + c / V : 0);
      float a = 0.f, b = 0.f;
      if (live)
        for (int r = lane; r < nrow; r += L) {
          const float2 o = e[r * q.sv];
          a += o.x;
          b += o.y;
        }
      a = lane_sum(a, L);
      b = lane_sum(b, L);
      if (live && lane == 0) {
        b *= st[2 * group_of(p, c) + 1];
        chan[c] = make_float2(a, b);
        if (p.N > 1) {
          p.cpart[(size_t)n * p.C + c0 + c] = make_float2(a, b);
        } else {
          if (p.dbeta) p.dbeta[c0 + c] = a + (p.acc_par ? p.dbeta[c0 + c] : 0.f);
          if (p.dgamma) p.dgamma[c0 + c] = b + (p.acc_par ? p.dgamma[c0 + c] : 0.f);
        }
      }
    }
  }
  __syncthreads();
  const int gs = nch / p.cg;
  {
    const int sh = lane_shift(gs, RES_NT), L = 1 << sh, lane = tid & (L - 1);
    for (int k = 0; k < gs; k += RES_NT >> sh) {
      const int g = k + (tid >> sh);
      float a = 0.f, b = 0.f;
      if (g < gs)
        for (int c = g * p.cg + lane; c < (g + 1) * p.cg; c += L) {
          const float w = p.gamma ? p.gamma[c0 + c] : 1.f;
          a = fmaf(w, chan[c].x, a);
          b = fmaf(w, chan[c].y, b);
        }
      a = lane_sum(a, L);
      b = lane_sum(b, L);
      if (g < gs && lane == 0) {
        const double inv = p.inv_count;
        gmean[g] = make_float2((float)(a * inv), (float)(b * inv));
      }
    }
  }
  __syncthreads();
  if (cnt == 0) return;
  float k0[V], k1[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int g = group_of(p, col * V + e);
    const float rs = st[2 * g + 1];
    k0[e] = -rs * gmean[g].x;
    k1[e] = -rs * rs * gmean[g].y;
  }
  T* po = (T*)p.out + row0 * p.o_ld + c0 + (size_t)col * V;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i < cnt) {
      float f[V], d[V], o[V];
      Lane<T, V>::cvt(rx[i], f);
      Lane<T, V>::cvt(rd[i], d);
      if (p.acc_dx) lane_load<T, V>(po + (size_t)i * q.rpb * p.o_ld, o);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float c = f[e] - mu[e];
        const float du = d[e] * gn_act_grad<Vec<T>::precise>(fmaf(ga[e], c, be[e]), act);
        const float g = fmaf(ga[e], du, fmaf(k1[e], c, k0[e]));
        d[e] = p.acc_dx ? o[e] + g : g;
      }
      Lane<T, V>::store(po + (size_t)i * q.rpb * p.o_ld, d);
    }
}

// ------------------------------------------------------------------------------------------------ host side
// Row chunks of one image in the streaming launches.  A function of the descriptor's sizes alone, so that the workspace does not depend on
// addresses: four workgroups per compute unit over the whole batch (eight: 8 x 6400 x 320 bf16 forward 49 instead of 35 us), and at least 8192
// values per chunk (2048 where that would leave fewer than 128 workgroups).  From 2^28 .. 2^29 values on (bf16, by C; fp32 half) there are more workgroups
// instead of longer ones: a thread then sums THREAD_ROWS rows in fp32, and a chunk whose first value dwarfs the rest keeps its M2 to THREAD_ROWS^2 half
// steps at worst (4e-3; with 8208 rows a thread 0.12 was measured).
constexpr int THREAD_ROWS = 256;
void gn_chunks(const plyolo_gn_desc* d, int* chunks, int* rows) {
  const int64_t all = (int64_t)d->N * d->HW;
  int64_t r = (all + 1023) / 1024;
  const int64_t values = all * d->C / 128, least = (min(max(values, (int64_t)2048), (int64_t)8192) + d->C - 1) / d->C;
  if (r < least) r = least;
  const int V = d->dtype == PLYOLO_BF16 ? 8 : 4, cols = min(d->C >= V ? cdiv(d->C, V) : d->C, 256);
  r = min(r, (int64_t)THREAD_ROWS * (256 / cols));
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
  // a launch has fewer than 2^32 threads: 1024 for every JOIN_I groups of an image, and for at most 128 blocks of channels
  PLY_CHECK_ARG((double)d->N * cdiv(d->groups, JOIN_I) < 4194304.0 - 128, "%s: too many images (%d)", who, d->N);
  PLY_CHECK_ARG(d->act >= PLYOLO_ACT_NONE && d->act <= PLYOLO_ACT_GELU, "%s: bad activation %d", who, d->act);
  PLY_CHECK_ARG(d->eps >= 0.f, "%s: eps must not be negative", who);
  PLY_CHECK_ARG(d->x_ld >= d->C, "%s: x_ld %d < C %d", who, d->x_ld, d->C);
  return 0;
}

size_t gn_ws_bytes(const plyolo_gn_desc* d) {
  int chunks, rows;
  gn_chunks(d, &chunks, &rows);
  return (size_t)d->N * (chunks * ((size_t)d->groups + d->C) + d->groups) * sizeof(float2);
}

GnP gn_params(const plyolo_gn_desc* d, void* ws) {
  GnP p{};
  p.N = d->N; p.HW = d->HW; p.C = d->C; p.G = d->groups; p.cg = d->C / d->groups; p.act = d->act;
  p.x_ld = d->x_ld; p.r_ld = d->r_ld; p.eps = d->eps;
  p.inv_cg = 1.0f / (float)p.cg;
  p.inv_count = 1.0 / ((double)p.HW * p.cg);
  gn_chunks(d, &p.chunks, &p.rows);
  p.gpart = (float2*)ws;
  p.cpart = p.gpart + (size_t)p.N * p.chunks * p.G;
  p.gmean = p.cpart + (size_t)p.N * p.chunks * p.C;
  return p;
}

// The resident split of the descriptor, or nv = 0 for the streaming launches.  A slice is a multiple of the least run of vectors that holds
// whole groups; it grows towards 128-byte row pieces as long as the batch still gives every compute unit a workgroup and the rows fit the
// registers (nv vectors a thread).  Measured, resident / streaming: the forward keeps its lead to the register limit when there are
// workgroups to fill the chip (32 x 6400 x 128 bf16, 25 vectors in a 512-thread workgroup and so 13 in the 1024-thread one that is launched:
// 38 / 42 us, cached 29 / 41; 32 x 1600 x 256: 18.5 / 32), one image on a few workgroups loses it beyond 12 vectors (1 x 6400 x 128, 13: 15.1
// / 14.7).  The backward holds two operands and has nothing to hide narrow row pieces behind: 16 vectors in pieces of 64 bytes and more
// (32 x 1600 x 256, sv 4: 29 / 42; 16 x 1600 x 640, sv 5: 40 / 49), 8 in narrower ones (32 x 6400 x 128, sv 1, nv 13: 90 / 68) and on few
// workgroups.
struct ResPlan { int sv, slices, rpb, nv, nt; };
ResPlan res_plan(const plyolo_gn_desc* d, int V, bool bwd) {
  ResPlan r{};
  const int cg = d->C / d->groups;
  int least = 1;
  while ((least * V) % cg != 0 && least * V < d->C) ++least;
  const int cv = d->C / V;
  if (least * V > 2048 || least > RES_NT || cv % least != 0) return r;      // (LDS: two floats per channel of the slice)
  const int esz = V == 1 ? 8 : 1;                     // element lanes: count eight of them as a vector
  for (int sv = least; sv <= cv && sv <= 8 * esz + least; sv += least) {
    if (cv % sv != 0 || sv > RES_NT) continue;
    const int64_t wgs = (int64_t)d->N * (cv / sv);
    if (wgs >= 4194304) continue;      // (a launch has fewer than 2^32 threads)
    const int rpb = RES_NT / sv, nv = (d->HW + rpb - 1) / rpb;
    if (nv > (V == 1 ? 16 : wgs < 64 ? (bwd ? 8 : 12) : bwd ? (sv >= 4 ? 16 : 8) : 32)) continue;
    if (sv > least && wgs < 256) break;
    r.sv = sv; r.slices = cv / sv; r.rpb = rpb; r.nv = nv;
  }
  r.nt = RES_NT;
  if (!bwd && r.nv > 16) {      // twice the threads with half the vectors each
    r.nt = 2 * RES_NT;
    r.rpb = r.nt / r.sv;
    r.nv = (d->HW + r.rpb - 1) / r.rpb;
  }
  return r;
}

#define GN_RES_FWD(T, V, nv, ACT)                                                                      \
  (rp.nt != RES_NT ? gn_res_fwd_kernel<T, V, 16, ACT, 2 * RES_NT> : (nv) <= 2 ? gn_res_fwd_kernel<T, V, 2, ACT, RES_NT> : (nv) <= 4 ? gn_res_fwd_kernel<T, V, 4, ACT, RES_NT>           \
   : (nv) <= 8 ? gn_res_fwd_kernel<T, V, 8, ACT, RES_NT> : gn_res_fwd_kernel<T, V, 16, ACT, RES_NT>)
#define GN_RES_BWD(T, V, nv, ACT) \
  ((nv) <= 2 ? gn_res_bwd_kernel<T, V, 2, ACT> : (nv) <= 4 ? gn_res_bwd_kernel<T, V, 4, ACT>           \
   : (nv) <= 8 ? gn_res_bwd_kernel<T, V, 8, ACT> : gn_res_bwd_kernel<T, V, 16, ACT>)
#define GN_RES_DISPATCH(dtype, wide, act, NAME, ELEM, nv)                                                                        \
  ((dtype) == PLYOLO_BF16 ? ((wide) ? ((act) == PLYOLO_ACT_SILU ? NAME(bf16_t, 8, nv, PLYOLO_ACT_SILU) : NAME(bf16_t, 8, nv, -1)) \
                                    : ELEM(bf16_t))                                                                             \
                          : ((wide) ? NAME(float, 4, nv, -1) : ELEM(float)))
#define GN_RES_FWD1(T) gn_res_fwd_kernel<T, 1, 16, -1, RES_NT>
#define GN_RES_BWD1(T) gn_res_bwd_kernel<T, 1, 16, -1>

// rows of whole vectors, rows with a cut last vector, rows of fewer channels than a vector
#define GN_DISPATCH(dtype, whole, wide, act, KERN)                                                                                       \
  ((dtype) == PLYOLO_BF16                                                                                                                 \
       ? ((whole)  ? ((act) == PLYOLO_ACT_SILU ? KERN<bf16_t, 8, PLYOLO_ACT_SILU, false> : KERN<bf16_t, 8, -1, false>)                      \
          : (wide) ? ((act) == PLYOLO_ACT_SILU ? KERN<bf16_t, 8, PLYOLO_ACT_SILU, true> : KERN<bf16_t, 8, -1, true>)                        \
                   : KERN<bf16_t, 1, -1, false>)                                                                                          \
       : ((whole) ? KERN<float, 4, -1, false> : (wide) ? KERN<float, 4, -1, true> : KERN<float, 1, -1, false>))

void join_bwd(const GnP& p, int npar, int nmean, int parts, hipStream_t s) {
  if (parts <= JOIN_FEW) hipLaunchKernelGGL(gn_join_bwd_kernel<256>, dim3((unsigned)(npar + nmean)), dim3(256), 0, s, p, npar, parts);
  else hipLaunchKernelGGL(gn_join_bwd_kernel<1024>, dim3((unsigned)(npar + nmean)), dim3(1024), 0, s, p, npar, parts);
}

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
  const bool wide = d->C >= V, whole = d->C % V == 0;
  plyolo::annotate("gn_act_fwd", 0.0, (double)p.N * p.HW * p.C * es * (res ? 3.0 : 2.0));
  const ResPlan rp = res_plan(d, whole ? V : 1, false);
  if (rp.nv) {
    ResP q{};
    q.g = p; q.sv = rp.sv; q.slices = rp.slices; q.rpb = rp.rpb;
    const int nch = rp.sv * (whole ? V : 1);
    const size_t lds = (size_t)(rp.nt * (whole ? V : 1) + nch + nch / p.cg) * sizeof(float2);
    return plyolo::submit(stream, [=](hipStream_t s) -> hipError_t {
      auto k = GN_RES_DISPATCH(dtype, whole, act, GN_RES_FWD, GN_RES_FWD1, rp.nv);
      if (hipError_t e = plyolo::ensure_dynamic_lds((const void*)k, lds); e != hipSuccess) return e;
      hipLaunchKernelGGL(k, dim3((unsigned)p.N * rp.slices), dim3(rp.nt), lds, s, q);
      return hipGetLastError();
    });
  }
  return plyolo::submit(stream, [=](hipStream_t s) -> hipError_t {
    auto ks = dtype == PLYOLO_BF16 ? (whole ? gn_stats_kernel<bf16_t, 8, false> : wide ? gn_stats_kernel<bf16_t, 8, true> : gn_stats_kernel<bf16_t, 1, false>)
                                   : (whole ? gn_stats_kernel<float, 4, false> : wide ? gn_stats_kernel<float, 4, true> : gn_stats_kernel<float, 1, false>);
    auto ka = GN_DISPATCH(dtype, whole, wide, act, gn_apply_kernel);
    const dim3 grid((unsigned)p.N * p.chunks), blk(256);
    const bool few = p.chunks <= JOIN_FEW;
    auto kj = dtype == PLYOLO_BF16 ? (few ? gn_join_fwd_kernel<bf16_t, 256> : gn_join_fwd_kernel<bf16_t, 1024>)
                                   : (few ? gn_join_fwd_kernel<float, 256> : gn_join_fwd_kernel<float, 1024>);
    hipLaunchKernelGGL(ks, grid, blk, (size_t)p.C * sizeof(float2), s, p);
    hipLaunchKernelGGL(kj, dim3((unsigned)p.N * cdiv(p.G, JOIN_I)), dim3(few ? 256 : 1024), 0, s, p);
    hipLaunchKernelGGL(ka, grid, blk, 0, s, p);
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
  const bool wide = d->C >= V, whole = d->C % V == 0;
  plyolo::annotate("gn_act_bwd", 0.0, (double)p.N * p.HW * p.C * es * (accumulate_dx ? 4.0 : 3.0));
  const ResPlan rp = res_plan(d, whole ? V : 1, true);
  if (rp.nv) {
    ResP q{};
    q.g = p; q.sv = rp.sv; q.slices = rp.slices; q.rpb = rp.rpb;
    const int nch = rp.sv * (whole ? V : 1);
    const size_t lds = (size_t)(nch + nch / p.cg) * sizeof(float2);
    return plyolo::submit(stream, [=](hipStream_t s) -> hipError_t {
      auto k = GN_RES_DISPATCH(dtype, whole, act, GN_RES_BWD, GN_RES_BWD1, rp.nv);
      hipLaunchKernelGGL(k, dim3((unsigned)p.N * rp.slices), dim3(RES_NT), lds, s, q);
      if (p.N > 1 && (p.dgamma || p.dbeta)) join_bwd(p, cdiv(p.C, JOIN_I), 0, p.N, s);
      return hipGetLastError();
    });
  }
  return plyolo::submit(stream, [=](hipStream_t s) -> hipError_t {
    auto ks = GN_DISPATCH(dtype, whole, wide, act, gn_bwd_sums_kernel);
    auto kd = GN_DISPATCH(dtype, whole, wide, act, gn_bwd_dx_kernel);
    const unsigned nblk = (unsigned)p.N * p.chunks;
    const int npar = (p.dgamma || p.dbeta) ? cdiv(p.C, JOIN_I) : 0;
    hipLaunchKernelGGL(ks, dim3(nblk), dim3(256), (size_t)p.C * sizeof(float2), s, p);
    join_bwd(p, npar, p.N * cdiv(p.G, JOIN_I), p.N * p.chunks, s);
    hipLaunchKernelGGL(kd, dim3(nblk), dim3(256), 0, s, p);
    return hipGetLastError();
  });
}

}  // extern "C"
