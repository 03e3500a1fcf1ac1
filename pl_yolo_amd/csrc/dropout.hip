// Dropout whose mask is never stored: a counter-based generator gives the random word of element i from (seed, step, site, i), so the
// backward forms the forward's mask again instead of reading it.
//
//     out = (keep(i) ? x / (1 - p) : 0) + res,   keep(i) = word(i) >> 8 >= round(p * 2^24),   i = m * C + c
//
// word(i) = word i % 4 of Philox4x32-7 at counter (i / 4, step, site) under the seed's halves as key (Salmon, Moraes, Dror, Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", SC 2011).  One counter serves four elements.  Seven rounds are the fewest the authors report as
// passing BigCrush; a round is two 32 x 32 -> 64 bit products (the part's quarter-rate multiplier) and six xors per four elements.
//
// The stream is HBM's: x (and res) in, out out.  One thread takes whole 16-byte vectors (8 bf16: two counters; 4 fp32: one); the element
// index of vector v is v * V whatever the row pitch, so only the address needs the row.
#include <math.h>

#include "common.h"

namespace {

struct DropP {
  const void* x;
  const void* res;      // NULL: none
  void* out;
  const uint64_t* rng;
  size_t total;         // M * C elements
  int C, x_ld, r_ld, o_ld;
  unsigned site, thr;   // keep <=> word >= thr (24 significant bits), unless none
  int none;             // p = 1
  int accumulate;
  float scale;
};

DEVINL void philox4x32_7(unsigned c0, unsigned c1, unsigned c2, unsigned c3, unsigned k0, unsigned k1, unsigned (&w)[4]) {
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
    c1 = (unsigned)b;
    c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
    c3 = (unsigned)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

struct Key { unsigned k0, k1, step; };
DEVINL Key load_key(const uint64_t* rng) {
  const uint64_t seed = rng[0], step = rng[1];
  return Key{(unsigned)seed, (unsigned)(seed >> 32), (unsigned)step};
}

// one vector of V elements starting at element v * V: f <- dropped f (+ r)
template <int V> DEVINL void drop_vec(const DropP& p, const Key& key, size_t v, float* f) {
#pragma unroll
  for (int j = 0; j < V / 4; ++j) {
    const size_t q = v * (V / 4) + j;
    unsigned w[4];
    philox4x32_7((unsigned)q, (unsigned)(q >> 32), key.step, p.site, key.k0, key.k1, w);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[4 * j + e] = (w[e] >= p.thr && !p.none) ? f[4 * j + e] * p.scale : 0.f;
  }
}

constexpr int DROP_U = 2;   // vectors in flight per thread

// HBM's copy rate: 204800 x 128 bf16 with shortcut 30 us, 5.2 TB/s (operands from HBM; 25 us from the last-level cache).
// whole 16-byte vectors; FLAT: no pitch anywhere (one long row, any C), else C is a multiple of V
template <typename T, bool FLAT> __global__ __launch_bounds__(256) void dropout_kernel(const DropP p) {
  constexpr int V = Vec<T>::N;
  const Key key = load_key(p.rng);
  const size_t nvec = p.total / V;
  const unsigned cv = (unsigned)(p.C / V);
  const size_t v0 = (size_t)blockIdx.x * (256 * DROP_U) + threadIdx.x;
  size_t xo[DROP_U], ro[DROP_U], oo[DROP_U];
  typename Vec<T>::raw_t xr[DROP_U], rr[DROP_U];
#pragma unroll
  for (int u = 0; u < DROP_U; ++u) {
    const size_t v = v0 + (size_t)u * 256;
    if (v >= nvec) continue;
    if (FLAT) {
      xo[u] = ro[u] = oo[u] = v * V;
    } else {
      const size_t m = nvec <= 0xffffffffu ? (size_t)((unsigned)v / cv) : v / cv;
      const size_t c = (v - m * cv) * V;
      xo[u] = m * p.x_ld + c;
      ro[u] = m * p.r_ld + c;
      oo[u] = m * p.o_ld + c;
    }
    xr[u] = Vec<T>::load_raw((const T*)p.x + xo[u]);
    if (p.res) rr[u] = Vec<T>::load_raw((const T*)p.res + ro[u]);
    else if (p.accumulate) rr[u] = Vec<T>::load_raw((const T*)p.out + oo[u]);
  }
#pragma unroll
  for (int u = 0; u < DROP_U; ++u) {
    const size_t v = v0 + (size_t)u * 256;
    if (v >= nvec) continue;
    float f[V], r[V];
    Vec<T>::cvt(xr[u], f);
    drop_vec<V>(p, key, v, f);
    if (p.res || p.accumulate) {
      Vec<T>::cvt(rr[u], r);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] += r[e];
    }
    Vec<T>::store((T*)p.out + oo[u], f);
  }
  if (FLAT && blockIdx.x == 0) {      // the elements behind the last whole vector
    const size_t i = nvec * V + threadIdx.x;
    if (i < p.total) {
      unsigned w[4];
      philox4x32_7((unsigned)(i / 4), (unsigned)((i / 4) >> 32), key.step, p.site, key.k0, key.k1, w);
      const unsigned e = (unsigned)i & 3, word = e == 0 ? w[0] : e == 1 ? w[1] : e == 2 ? w[2] : w[3];
      float f = (word >= p.thr && !p.none) ? ActT<T>::ld((const T*)p.x + i) * p.scale : 0.f;
      if (p.res) f += ActT<T>::ld((const T*)p.res + i);
      else if (p.accumulate) f += ActT<T>::ld((const T*)p.out + i);
      ActT<T>::st((T*)p.out + i, f);
    }
  }
}

// four consecutive elements
template <typename T> struct Four;
template <> struct Four<bf16_t> {
  typedef unsigned type __attribute__((ext_vector_type(2)));
  static DEVINL void cvt(const type v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x << 16);
    f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16);
    f[3] = __uint_as_float(v.y & 0xffff0000u);
  }
  static DEVINL type pack(const float (&f)[4]) { return type{pack2bf(f[0], f[1]), pack2bf(f[2], f[3])}; }
};
template <> struct Four<float> {
  typedef f32x4 type;
  static DEVINL void cvt(const f32x4 v, float (&f)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = v[e];
  }
  static DEVINL f32x4 pack(const float (&f)[4]) { return f32x4{f[0], f[1], f[2], f[3]}; }
};

// any C, pitch and alignment: one thread per counter, one by one where its four elements are of two rows (20000 x 613 bf16 with shortcut, pitch
// 616: 20 us; every element by itself 28; the same without a pitch, in whole vectors, 14)
template <typename T> __global__ __launch_bounds__(256) void dropout_any_kernel(const DropP p) {
  const Key key = load_key(p.rng);
  const size_t q = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (q * 4 >= p.total) return;
  unsigned w[4];
  philox4x32_7((unsigned)q, (unsigned)(q >> 32), key.step, p.site, key.k0, key.k1, w);
  size_t m = p.total <= 0xffffffffu ? (size_t)((unsigned)(q * 4) / (unsigned)p.C) : q * 4 / p.C;
  int c = (int)(q * 4 - m * p.C);
  if (c + 4 <= p.C) {      // the whole counter in one row: 8 or 16 bytes at any element address
    typedef typename Four<T>::type __attribute__((aligned(sizeof(T)))) any4;
    T* o = (T*)p.out + m * p.o_ld + c;
    float f[4], r[4];
    Four<T>::cvt(*(const any4*)((const T*)p.x + m * p.x_ld + c), f);
    if (p.res) Four<T>::cvt(*(const any4*)((const T*)p.res + m * p.r_ld + c), r);
    else if (p.accumulate) Four<T>::cvt(*(const any4*)o, r);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[e] = (w[e] >= p.thr && !p.none) ? f[e] * p.scale : 0.f;
      if (p.res || p.accumulate) f[e] += r[e];
    }
    *(any4*)o = Four<T>::pack(f);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (q * 4 + e < p.total) {
      T* o = (T*)p.out + m * p.o_ld + c;
      float f = (w[e] >= p.thr && !p.none) ? ActT<T>::ld((const T*)p.x + m * p.x_ld + c) * p.scale : 0.f;
      if (p.res) f += ActT<T>::ld((const T*)p.res + m * p.r_ld + c);
      else if (p.accumulate) f += ActT<T>::ld(o);
      ActT<T>::st(o, f);
    }
    if (++c == p.C) { c = 0; ++m; }
  }
}

__global__ void rng_next_kernel(uint64_t* state, uint64_t* out) {
  const uint64_t seed = state[0], step = state[1];
  out[0] = seed;
  out[1] = step;
  state[1] = step + 1;
}

int dropout_submit(const char* who, int dtype, int M, int C, const void* x, int x_ld, float pr, const uint64_t* rng, unsigned site,
                   const void* res, int r_ld, void* out, int o_ld, int accumulate, void* stream) {
  PLY_CHECK_ARG(dtype == PLYOLO_BF16 || dtype == PLYOLO_F32, "%s: bad dtype %d", who, dtype);
  PLY_CHECK_ARG(M > 0 && C > 0, "%s: non-positive dimension (M %d, C %d)", who, M, C);
  PLY_CHECK_ARG(x && out && rng, "%s: null operand", who);
  PLY_CHECK_ARG(pr >= 0.f && pr <= 1.f, "%s: p must be in [0, 1]", who);
  PLY_CHECK_ARG(x_ld >= C && o_ld >= C && (!res || r_ld >= C), "%s: a row pitch is smaller than C = %d", who, C);
  const size_t es = dtype == PLYOLO_BF16 ? 2 : 4;
  PLY_CHECK_ARG(((size_t)x | (size_t)out | (size_t)res) % es == 0 && (size_t)rng % 8 == 0, "%s: misaligned operand", who);
  DropP p{};
  p.x = x; p.res = res; p.out = out; p.rng = rng;
  p.total = (size_t)M * C;
  p.C = C; p.x_ld = x_ld; p.r_ld = r_ld; p.o_ld = o_ld;
  p.site = site;
  const unsigned t24 = (unsigned)rint((double)pr * 16777216.0);
  p.none = t24 >= 16777216u;
  p.thr = p.none ? 0xffffffffu : t24 << 8;
  p.scale = p.none ? 0.f : (float)(1.0 / (1.0 - (double)pr));
  p.accumulate = accumulate;
  const int V = dtype == PLYOLO_BF16 ? 8 : 4;
  const bool aligned = ((size_t)x | (size_t)out | (size_t)res) % 16 == 0;
  const bool flat = aligned && (M == 1 || (x_ld == C && o_ld == C && (!res || r_ld == C)));
  const bool wide = aligned && C % V == 0 && x_ld % V == 0 && o_ld % V == 0 && (!res || r_ld % V == 0);
  const size_t per = (flat || wide) ? (size_t)V * 256 * DROP_U : (size_t)4 * 256;
  const size_t grid = cdivz(p.total, per);
  PLY_CHECK_ARG(grid < 16777216u, "%s: more than 2^24 workgroups", who);
  plyolo::annotate(who, 0.0, (double)p.total * es * (res || accumulate ? 3.0 : 2.0));
  return plyolo::submit(stream, [=](hipStream_t s) -> hipError_t {
    const dim3 g((unsigned)grid), b(256);
    if (dtype == PLYOLO_BF16) {
      auto k = flat ? dropout_kernel<bf16_t, true> : wide ? dropout_kernel<bf16_t, false> : dropout_any_kernel<bf16_t>;
      hipLaunchKernelGGL(k, g, b, 0, s, p);
    } else {
      auto k = flat ? dropout_kernel<float, true> : wide ? dropout_kernel<float, false> : dropout_any_kernel<float>;
      hipLaunchKernelGGL(k, g, b, 0, s, p);
    }
    return hipGetLastError();
  });
}

}  // namespace

extern "C" {

int plyolo_rng_next(uint64_t* state, uint64_t* out, void* stream) {
  PLY_CHECK_ARG(state && out && ((size_t)state | (size_t)out) % 8 == 0, "rng_next: null or misaligned state");
  plyolo::annotate("rng_next", 0.0, 32.0);
  return plyolo::submit(stream, [=](hipStream_t s) -> hipError_t {
    hipLaunchKernelGGL(rng_next_kernel, dim3(1), dim3(1), 0, s, state, out);
    return hipGetLastError();
  });
}

int plyolo_dropout_fwd(int dtype, int M, int C, const void* x, int x_ld, float p, const uint64_t* rng, unsigned site, const void* res, int r_ld,
                       void* out, int o_ld, void* stream) {
  return dropout_submit("dropout_fwd", dtype, M, C, x, x_ld, p, rng, site, res, r_ld, out, o_ld, 0, stream);
}

int plyolo_dropout_bwd(int dtype, int M, int C, const void* dout, int d_ld, float p, const uint64_t* rng, unsigned site, void* dx, int dx_ld,
                       int accumulate, void* stream) {
  return dropout_submit("dropout_bwd", dtype, M, C, dout, d_ld, p, rng, site, nullptr, 0, dx, dx_ld, accumulate ? 1 : 0, stream);
}

}  // extern "C"
