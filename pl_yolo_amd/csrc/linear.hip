// Linear layer (1x1 convolution with bias) with activation and shortcut in its epilogue, forward and backward.
//
//   z = x . w^T + bias,  y = act(z) + res          x [M][K], w [N][K], y, z [M][N]
//   dz = dy act'(z),  dx = dz . w,  dw = dz^T . x,  db = sum over rows of dz
//
// All three products are one kernel body over two operands that are either contiguous along the contraction (KC: x and w of the forward,
// dz of dx) or along the output (RC: w of dx, dz and x of dw); an RC operand is transposed on its way out of LDS (ds_read_b64_tr_b16 in bf16).
// The product is formed as D = B . A^T, so that a lane of the MFMA result holds four consecutive COLUMNS of one output row: 8 bytes of bf16, put
// together to whole row pieces in LDS, or 16 of fp32, stored as they are.
//
// bf16: dz is rounded to bf16 once, as the operand of both matrix products (db sums it unrounded); dw has that rounding's noise beside its own.
//
// dw contracts over the rows of the batch: the rows are split over workgroups, every range leaves a private fp32 slab and the slabs are
// added in a fixed order.
//
// Times in this file are of whole calls in a captured graph that goes over three sets of operands in turn (more than the last-level cache
// holds comes from HBM), sizes M x K x N, forwards with z; "cached": over one set.  The profiler times kernels one by one, which
// can come out above their share of a stream (12800 x 2048 x 1024 78 us).
#include "common.h"

namespace {

enum { MODE_FWD = 0, MODE_DX = 1, MODE_DW = 2 };

struct LinP {
  const void* a;       // operand whose rows are output rows i
  const void* b;       // operand whose rows are output columns j
  void* out;           // y | dx | dw (one slab) or fp32 slabs
  void* z;             // forward: pre-activation out, or NULL
  const void* res;     // forward: shortcut, or NULL
  const float* bias;   // forward, or NULL
  int I, J, Kc;        // output rows, output columns, contraction length
  int a_ld, b_ld, o_ld, z_ld, r_ld;
  int act, accumulate;
  int vec4;            // blocks of the forward, slabs: four columns leave at once
  int nj, tiles;       // column tiles, all tiles of the output
  int ksteps;          // MODE_DW: contraction stages per slab
};

// ------------------------------------------------------------------------------------------------ bf16
constexpr int BK = 64;           // contraction elements per stage (and the unit that dw's row ranges are counted in)
typedef u32x4 __attribute__((aligned(2))) u32x4_any;     // 16 bytes at any element address
typedef f32x4 __attribute__((aligned(4))) f32x4_any;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
DEVINL s16x4 tr_read(const unsigned char* p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p); }

__device__ u32x4 zero_granule;   // where the lanes of a direct load that have nothing to fetch read from

// eight consecutive elements of which `n` >= 1 exist (the others are zero; the loads of a tail are all requested before one is used)
DEVINL u32x4 load8(const bf16_t* p, int n) {
  if (n >= 8) return *(const u32x4_any*)p;
  unsigned h[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = p[min(e, n - 1)];
  u32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (2 * e < n ? h[2 * e] : 0u) | (2 * e + 1 < n ? h[2 * e + 1] << 16 : 0u);
  return v;
}

// drops the first e (1 .. 7) of eight elements
DEVINL u32x4 shift_out(u32x4 v, int e) {
  uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
  if (e >= 4) { lo = hi; hi = 0; e -= 4; }
  if (e > 0) {
    lo = lo >> (16 * e) | hi << (64 - 16 * e);
    hi >>= 16 * e;
  }
  return u32x4{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32)};
}

DEVINL void store8(bf16_t* p, int n, u32x4 v) {
  if (n >= 8) {
    *(u32x4_any*)p = v;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = (bf16_t)(v[e >> 1] >> (16 * (e & 1)));
  }
}

DEVINL int xcd_contiguous(int id, int n) {      // hardware deals workgroup ids round robin over the 8 XCDs: give each a contiguous range
  const int q = n >> 3, r = n & 7, x = id & 7;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (id >> 3);
}

// Output tile and (MODE_DW) contraction slab of a workgroup.  Neighbours read the same rows, so they get neighbouring ids on one XCD and its L2
// serves all but the first of them: column tiles of one row tile, and all tiles of one slab.
struct Place { int i0, j0, slab; };
template <int TI, int TJ> DEVINL Place place(const LinP& p, int block, int blocks) {
  const int id = xcd_contiguous(block, blocks), tile = id % p.tiles;
  return Place{tile / p.nj * TI, tile % p.nj * TJ, id / p.tiles};
}

// One operand tile: T rows (output index) x K contraction elements, NT threads.
// KC image: [T][K] elements, rows of K / 8 16-byte granules, granule g of row r at position g ^ f(r).
// RC image: [K][T] elements, rows of T / 16 32-byte segments, segment s of row k at position s ^ f(k): the 16 rows that one transposed read
// of a wave touches spread over all banks.
// DIRECT: whole granules at 16-byte addresses go to LDS without passing registers (a lane's destination is fixed by the instruction, so the
// swizzle is applied to its source); otherwise through registers: a granule that a row's end cuts is fetched as the row's last eight elements
// and shifted on its way to LDS, so that no request waits for another (rows of fewer than eight elements: one by one).
template <bool RC, int T, int K, int NT, bool DIRECT> struct Tile {
  static constexpr int NG = (T * K / 8 + NT - 1) / NT;      // 16-byte granules per thread (the last of them: whole waves only)
  static constexpr int BYTES = T * K * 2, KG = K / 8, TG = T / 8;
  static_assert(T * K / 8 % (DIRECT ? 64 : NT) == 0, "a wave requests whole granules or none");
  static DEVINL bool mine(int u) { return (u + 1) * NT * 8 <= T * K || (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 64 < T * K / 8 - u * NT; }
  static DEVINL int swz_k(int k) { return T >= 128 ? (k & 3) | ((k >> 1) & 4) : (k & 3); }
  static DEVINL int swz_r(int r) { return K == 64 ? r & 7 : (r >> 1) & 3; }
  const bf16_t* src[NG];     // granule u at contraction 0 of the workgroup (NULL: its row does not exist)
  int kof[NG];               // its contraction offset inside a stage
  u32x4 v[DIRECT ? 1 : NG];
  int len[DIRECT ? 1 : NG];  // RC: elements of the granule that exist
  int cut[DIRECT ? 1 : NG];  // of the granule in v: elements to shift out
  bool few;                  // rows of fewer than eight elements

  // clen: contraction elements of the whole operand
  DEVINL void init(const bf16_t* base, int ld, int row0, int rows, int kbeg, int clen) {
    few = (RC ? rows : clen) < 8;
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      const int idx = threadIdx.x + u * NT;
      if (RC) {
        const int k = idx / TG, pos = idx % TG;
        const int g = DIRECT ? ((((pos >> 1) ^ swz_k(k)) << 1) | (pos & 1)) : pos;
        const int r = row0 + g * 8;
        kof[u] = k;
        src[u] = r < rows ? base + (size_t)(kbeg + k) * ld + r : nullptr;
        if (!DIRECT) len[u] = rows - r;
      } else {
        const int r = row0 + idx / KG, pos = idx % KG, g = DIRECT ? pos ^ swz_r(idx / KG) : pos;
        kof[u] = g * 8;
        src[u] = r < rows ? base + (size_t)r * ld + kbeg + g * 8 : nullptr;
      }
    }
  }
  // the stage that starts `k` elements behind kbeg, `left` elements of the contraction are left there (none: zeros)
  DEVINL void request(unsigned char* img, size_t k, int ld, int left) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      const bf16_t* q = src[u] + (RC ? k * ld : k);
      const bool ok = src[u] != nullptr && kof[u] < left;
      if (DIRECT) {
        const void* g = ok ? (const void*)q : (const void*)&zero_granule;
        if (mine(u)) __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                         (__attribute__((address_space(3))) void*)(img + (u * NT + wave * 64) * 16), 16, 0, 0);
      } else {
        const int w = DIRECT ? 0 : u, n = RC ? len[w] : left - kof[u];
        cut[w] = ok && n < 8 && !few ? 8 - n : 0;
        if (few) v[w] = ok ? load8(q, n) : u32x4{0u, 0u, 0u, 0u};
        else v[w] = *(ok ? (const u32x4_any*)(q - cut[w]) : (const u32x4_any*)&zero_granule);
      }
    }
  }
  DEVINL void commit(unsigned char* img) {
    if (DIRECT) return;
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      const int idx = threadIdx.x + u * NT;
      if (cut[DIRECT ? 0 : u]) v[DIRECT ? 0 : u] = shift_out(v[DIRECT ? 0 : u], cut[DIRECT ? 0 : u]);
      if (RC) {
        const int k = idx / TG, g = idx % TG;
        *(u32x4*)(img + k * (T * 2) + (((g >> 1) ^ swz_k(k)) << 5) + ((g & 1) << 4)) = v[DIRECT ? 0 : u];
      } else {
        const int r = idx / KG, g = idx % KG;
        *(u32x4*)(img + r * (K * 2) + ((g ^ swz_r(r)) << 4)) = v[DIRECT ? 0 : u];
      }
    }
  }
  // fragment of 16 output indices starting at r0, contraction elements 32 kk .. 32 kk + 31
  static DEVINL s16x8 frag(const unsigned char* img, int r0, int kk) {
    const int lane = threadIdx.x & 63, g4 = lane >> 4, i16 = lane & 15;
    if (RC) {
      const int k = kk * 32 + 8 * g4 + (i16 >> 2), seg = r0 >> 4;
      const unsigned char* p = img + k * (T * 2) + ((seg ^ swz_k(k)) << 5) + ((i16 & 3) << 3);
      const s16x4 lo = tr_read(p), hi = tr_read(p + 4 * (T * 2));       // (swz_k(k + 4) == swz_k(k))
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    const int r = r0 + i16, g = kk * 4 + g4;
    return *(const s16x8*)(img + r * (K * 2) + ((g ^ swz_r(r)) << 4));
  }
};

// HEAVY: hswish / GELU (their code stays out of the other instances)
template <bool HEAVY> DEVINL void act4(f32x4& v, int act) {
  if (!HEAVY && act == PLYOLO_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = act_fwd_core(v[e], PLYOLO_ACT_SILU);
  } else if (HEAVY || act != PLYOLO_ACT_NONE) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = HEAVY ? act_fwd(v[e], act) : act_fwd_core(v[e], act);
  }
}

// forward: four consecutive columns j.. of output row i; nv of them exist
template <bool HEAVY> DEVINL void store4(const LinP& p, int i, int j, f32x4 v, const f32x4 bias) {
  const int nv = p.J - j;
  if (i >= p.I || nv <= 0) return;
  const bool whole = p.vec4 && nv >= 4;
  v += bias;
  if (p.z) {
    bf16_t* z = (bf16_t*)p.z + (size_t)i * p.z_ld + j;
    if (whole) *(uint2*)z = make_uint2(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]));
    else
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < nv) z[e] = f2bf(v[e]);
  }
  act4<HEAVY>(v, p.act);
  bf16_t* o = (bf16_t*)p.out + (size_t)i * p.o_ld + j;
  const bf16_t* r = p.res ? (const bf16_t*)p.res + (size_t)i * p.r_ld + j : nullptr;
  if (whole) {
    if (r) {
      const uint2 t = *(const uint2*)r;
      v[0] += __uint_as_float(t.x << 16);
      v[1] += __uint_as_float(t.x & 0xffff0000u);
      v[2] += __uint_as_float(t.y << 16);
      v[3] += __uint_as_float(t.y & 0xffff0000u);
    }
    *(uint2*)o = make_uint2(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < nv) o[e] = f2bf(r ? v[e] + bf2f(r[e]) : v[e]);
  }
}

// the bias of columns j .. j + 3 (zeros where there is none)
template <int MODE> DEVINL f32x4 bias4(const LinP& p, int j) {
  f32x4 b = {0.f, 0.f, 0.f, 0.f};
  if (MODE == MODE_FWD && p.bias) {
    if (j + 4 <= p.J) {
      b = *(const f32x4_any*)(p.bias + j);
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (j + e < p.J) b[e] = p.bias[j + e];
    }
  }
  return b;
}
// ... of a wave's columns, requested in front of the contraction
template <int MODE, int FB> struct Bias {
  f32x4 v[MODE == MODE_FWD ? FB : 1];
  DEVINL Bias(const LinP& p, int j0) {
    if (MODE == MODE_FWD) {
#pragma unroll
      for (int b = 0; b < FB; ++b) v[b] = bias4<MODE>(p, j0 + b * 16 + 4 * ((threadIdx.x & 63) >> 4));
    }
  }
};

// Rows leave (and the shortcut's rows, or dx's own for an accumulation, arrive) through LDS: a lane of the MFMA result holds 8 bytes of a row,
// written as they are they would cost four times the requests of whole row pieces.  z and y take the same image one after the other: less LDS
// is one workgroup per compute unit more.
template <int TI, int TJ> constexpr size_t out_bytes() { return (size_t)TI * (TJ * 2 + 16); }

template <int TI, int TJ, int NT> DEVINL void rows_out(const LinP& p, const unsigned char* img, int i0, int j0, bf16_t* out, int ld) {
  constexpr int PITCH = TJ * 2 + 16, RV = TJ / 8;
#pragma unroll 4
  for (int idx = threadIdx.x; idx < TI * RV; idx += NT) {
    const int r = idx / RV, c = idx % RV * 8, n = p.J - j0 - c;
    if (i0 + r < p.I && n > 0) store8(out + (size_t)(i0 + r) * ld + j0 + c, n, *(const u32x4*)(img + r * PITCH + c * 2));
  }
}

template <int MODE, int TI, int TJ, int NT, int WI, int WJ, bool HEAVY>
DEVINL void tile_out(const LinP& p, unsigned char* img, int i0, int j0, const int wi, const int wj, f32x4 (&acc)[WI / 16][WJ / 16],
                     const Bias<MODE, WJ / 16>& bias) {
  constexpr int PITCH = TJ * 2 + 16, RV = TJ / 8, FA = WI / 16, FB = WJ / 16;
  const int lane = threadIdx.x & 63, at0 = (wi + (lane & 15)) * PITCH + (wj + 4 * (lane >> 4)) * 2;
  __syncthreads();
  if (MODE == MODE_FWD) {
#pragma unroll
    for (int a = 0; a < FA; ++a)
#pragma unroll
      for (int b = 0; b < FB; ++b) acc[a][b] += bias.v[b];
    if (p.z) {
#pragma unroll
      for (int a = 0; a < FA; ++a)
#pragma unroll
        for (int b = 0; b < FB; ++b)
          *(uint2*)(img + at0 + a * 16 * PITCH + b * 32) = make_uint2(pack2bf(acc[a][b][0], acc[a][b][1]), pack2bf(acc[a][b][2], acc[a][b][3]));
      __syncthreads();
      rows_out<TI, TJ, NT>(p, img, i0, j0, (bf16_t*)p.z, p.z_ld);
      __syncthreads();
    }
  }
  const bf16_t* rows = MODE == MODE_FWD ? (const bf16_t*)p.res : p.accumulate ? (const bf16_t*)p.out : nullptr;
  if (rows) {
    const int ld = MODE == MODE_FWD ? p.r_ld : p.o_ld;
    for (int idx = threadIdx.x; idx < TI * RV; idx += NT) {
      const int r = idx / RV, c = idx % RV * 8;
      if (i0 + r < p.I && j0 + c < p.J) *(u32x4*)(img + r * PITCH + c * 2) = load8(rows + (size_t)(i0 + r) * ld + j0 + c, p.J - j0 - c);
    }
    __syncthreads();
  }
#pragma unroll
  for (int a = 0; a < FA; ++a)
#pragma unroll
    for (int b = 0; b < FB; ++b) {
      unsigned char* at = img + at0 + a * 16 * PITCH + b * 32;
      f32x4 v = acc[a][b];
      if (MODE == MODE_FWD) act4<HEAVY>(v, p.act);
      if (rows) {
        const uint2 t = *(const uint2*)at;
        v[0] += __uint_as_float(t.x << 16);
        v[1] += __uint_as_float(t.x & 0xffff0000u);
        v[2] += __uint_as_float(t.y << 16);
        v[3] += __uint_as_float(t.y & 0xffff0000u);
      }
      *(uint2*)at = make_uint2(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]));
    }
  __syncthreads();
  rows_out<TI, TJ, NT>(p, img, i0, j0, (bf16_t*)p.out, p.o_ld);
}

// fp32 partial sums of a wave's block into its slab
template <int WI, int WJ> DEVINL void slab_out(const LinP& p, int slab, int i0, int j0, f32x4 (&acc)[WI / 16][WJ / 16]) {
  const int lane = threadIdx.x & 63;
  float* out = (float*)p.out + (size_t)slab * p.I * p.J;
#pragma unroll
  for (int b = 0; b < WJ / 16; ++b) {
    const int j = j0 + b * 16 + 4 * (lane >> 4), n = p.J - j;
#pragma unroll
    for (int a = 0; a < WI / 16; ++a) {
      const int i = i0 + a * 16 + (lane & 15);
      if (i >= p.I || n <= 0) continue;
      float* o = out + (size_t)i * p.J + j;
      if (p.vec4 && n >= 4) {
        *(f32x4*)o = acc[a][b];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < n) o[e] = acc[a][b][e];
      }
    }
  }
}

// Any size, pitch and alignment: TI x TJ tile, four waves of TI / 2 x TJ / 2, operands through registers into two LDS images, one barrier per
// stage: stage s + 1 is requested behind the barrier of stage s and lands under its MFMAs.  12800 x 2047 x 1023 126 us, 427 TFLOP/s.
template <int MODE, int TI, int TJ, bool HEAVY> DEVINL void any_tile(const LinP& p, int block, int blocks) {
  constexpr bool ARC = MODE == MODE_DW, BRC = MODE != MODE_FWD;
  typedef Tile<ARC, TI, BK, 256, false> TA;
  typedef Tile<BRC, TJ, BK, 256, false> TB;
  constexpr int FA = TI / 32, FB = TJ / 32, STAGE = TA::BYTES + TB::BYTES;
  extern __shared__ __align__(16) unsigned char smem[];
  const Place at = place<TI, TJ>(p, block, blocks);
  const int i0 = at.i0, j0 = at.j0;
  const int wave = threadIdx.x >> 6, wi = (wave >> 1) * (TI / 2), wj = (wave & 1) * (TJ / 2);
  const int kbeg = at.slab * p.ksteps * BK;
  const int klen = (MODE == MODE_DW ? min(p.Kc, kbeg + p.ksteps * BK) : p.Kc) - kbeg;
  f32x4 acc[FA][FB];
#pragma unroll
  for (int a = 0; a < FA; ++a)
#pragma unroll
    for (int b = 0; b < FB; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  const Bias<MODE, FB> bias(p, j0 + wj);
  TA ta;
  TB tb;
  ta.init((const bf16_t*)p.a, p.a_ld, i0, p.I, kbeg, p.Kc);
  tb.init((const bf16_t*)p.b, p.b_ld, j0, p.J, kbeg, p.Kc);
  ta.request(smem, 0, p.a_ld, klen);
  tb.request(smem, 0, p.b_ld, klen);
  int buf = 0;
  for (int k0 = 0; k0 < klen; k0 += BK, buf ^= 1) {
    unsigned char *ia = smem + buf * STAGE, *ib = ia + TA::BYTES;
    ta.commit(ia);
    tb.commit(ib);
    __syncthreads();      // image `buf` is whole; image buf ^ 1 was last read before every wave came here
    if (k0 + BK < klen) {
      ta.request(smem, k0 + BK, p.a_ld, klen - k0 - BK);
      tb.request(smem, k0 + BK, p.b_ld, klen - k0 - BK);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      s16x8 fa[FA], fb[FB];
#pragma unroll
      for (int a = 0; a < FA; ++a) fa[a] = TA::frag(ia, wi + a * 16, kk);
#pragma unroll
      for (int b = 0; b < FB; ++b) fb[b] = TB::frag(ib, wj + b * 16, kk);
#pragma unroll
      for (int a = 0; a < FA; ++a)
#pragma unroll
        for (int b = 0; b < FB; ++b)
          acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8*)&fb[b], *(const bf16x8*)&fa[a], acc[a][b], 0, 0, 0);
    }
  }
  if (MODE == MODE_DW) slab_out<TI / 2, TJ / 2>(p, at.slab, i0 + wi, j0 + wj, acc);
  else tile_out<MODE, TI, TJ, 256, TI / 2, TJ / 2, HEAVY>(p, smem, i0, j0, wi, wj, acc, bias);
}

// Aligned operands: NWI x NWJ waves of WI x WJ, ST LDS images of K contraction elements filled by direct loads, ST - 1 stages in flight: a
// stage's wait leaves the younger stages' loads outstanding.  One barrier per stage: behind it the image that was read in the stage before is
// free for the youngest request.  12800 x 2048 x 1024 64 us, 840 TFLOP/s (cached 58): the MFMAs of one round of tiles (44 % busy over the
// kernel), then 52 MB of stores.
template <int N> DEVINL void wait_and_meet() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

template <int MODE, int NWI, int NWJ, int WI, int WJ, int K, int ST, bool HEAVY> DEVINL void direct_tile(const LinP& p, int block, int blocks) {
  constexpr bool ARC = MODE == MODE_DW, BRC = MODE != MODE_FWD;
  constexpr int NT = 64 * NWI * NWJ, TI = NWI * WI, TJ = NWJ * WJ, FA = WI / 16, FB = WJ / 16;
  typedef Tile<ARC, TI, K, NT, true> TA;
  typedef Tile<BRC, TJ, K, NT, true> TB;
  constexpr int STAGE = TA::BYTES + TB::BYTES, LOADS = TA::NG + TB::NG;
  static_assert(ST >= 2 && ST <= 3 && (ST == 2 || (TI * K / 8 % NT == 0 && TJ * K / 8 % NT == 0)), "the waits below count a wave's loads");
  extern __shared__ __align__(16) unsigned char smem[];
  const Place at = place<TI, TJ>(p, block, blocks);
  const int i0 = at.i0, j0 = at.j0;
  const int wave = threadIdx.x >> 6, wi = wave / NWJ * WI, wj = wave % NWJ * WJ;
  const int kbeg = at.slab * p.ksteps * BK;
  const int klen = (MODE == MODE_DW ? min(p.Kc, kbeg + p.ksteps * BK) : p.Kc) - kbeg;
  f32x4 acc[FA][FB];
#pragma unroll
  for (int a = 0; a < FA; ++a)
#pragma unroll
    for (int b = 0; b < FB; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  const Bias<MODE, FB> bias(p, j0 + wj);
  TA ta;
  TB tb;
  ta.init((const bf16_t*)p.a, p.a_ld, i0, p.I, kbeg, p.Kc);
  tb.init((const bf16_t*)p.b, p.b_ld, j0, p.J, kbeg, p.Kc);
  for (int s = 0; s < ST - 1 && s * K < klen; ++s) {
    ta.request(smem + s * STAGE, s * K, p.a_ld, klen - s * K);
    tb.request(smem + s * STAGE + TA::BYTES, s * K, p.b_ld, klen - s * K);
  }
  int buf = 0;
  for (int k0 = 0; k0 < klen; k0 += K, buf = buf + 1 == ST ? 0 : buf + 1) {
    unsigned char *ia = smem + buf * STAGE, *ib = ia + TA::BYTES;
    const int behind = klen - k0;                  // stages requested behind this one: as many as there are, ST - 2 at most
    if (ST == 3 && behind > K) wait_and_meet<LOADS>();
    else wait_and_meet<0>();
    if (behind > (ST - 1) * K) {
      unsigned char* na = smem + (buf == 0 ? ST - 1 : buf - 1) * STAGE;
      ta.request(na, k0 + (ST - 1) * K, p.a_ld, behind - (ST - 1) * K);
      tb.request(na + TA::BYTES, k0 + (ST - 1) * K, p.b_ld, behind - (ST - 1) * K);
    }
#pragma unroll
    for (int kk = 0; kk < K / 32; ++kk) {
      s16x8 fa[FA], fb[FB];
#pragma unroll
      for (int b = 0; b < FB; ++b) fb[b] = TB::frag(ib, wj + b * 16, kk);
#pragma unroll
      for (int a = 0; a < FA; ++a) fa[a] = TA::frag(ia, wi + a * 16, kk);
#pragma unroll
      for (int a = 0; a < FA; ++a)
#pragma unroll
        for (int b = 0; b < FB; ++b)
          acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8*)&fb[b], *(const bf16x8*)&fa[a], acc[a][b], 0, 0, 0);
    }
    // the order of the stage: the first fragments, then some reads behind every row of MFMAs, so that no row waits for its own
    constexpr int RA = ARC ? 2 : 1, RB = BRC ? 2 : 1, ROWS = FA * (K / 32);      // (a transposed fragment is two LDS instructions)
    constexpr int FIRST = RB * FB + RA * 2, LATER = ((RB * FB + RA * FA) * (K / 32) - FIRST + ROWS - 1) / ROWS;
    __builtin_amdgcn_sched_group_barrier(0x100, FIRST, 0);
#pragma unroll
    for (int g = 0; g < ROWS; ++g) {
      __builtin_amdgcn_sched_group_barrier(0x008, FB, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, LATER, 0);
    }
  }
  if (MODE == MODE_DW) slab_out<WI, WJ>(p, at.slab, i0 + wi, j0 + wj, acc);
  else tile_out<MODE, TI, TJ, NT, WI, WJ, HEAVY>(p, smem, i0, j0, wi, wj, acc, bias);
}

template <int MODE, int T, bool HEAVY> __global__ __launch_bounds__(256) void linear_bf16_any_kernel(const LinP p) {
  any_tile<MODE, T, T, HEAVY>(p, blockIdx.x, gridDim.x);
}
template <int MODE, int NWI, int NWJ, int WI, int WJ, int K, int ST, bool HEAVY>
__global__ __launch_bounds__(64 * NWI * NWJ) void linear_bf16_kernel(const LinP p) {
  direct_tile<MODE, NWI, NWJ, WI, WJ, K, ST, HEAVY>(p, blockIdx.x, gridDim.x);
}
// Both products of the backward in one launch: workgroups [0, nw) form dw (few and long), the others dx (many and short) beside them.  Alone,
// neither keeps the memory system busy: 51200 x 256 x 256 19 + 20 us one after the other, 30 us together (the kernels alone, cached).
template <int T, bool DIRECT> __global__ __launch_bounds__(256) void linear_bf16_bwd_kernel(const LinP px, const LinP pw, const int nw) {
  const bool first = (int)blockIdx.x < nw;
  const int block = first ? blockIdx.x : blockIdx.x - nw, blocks = first ? nw : gridDim.x - nw;
  if constexpr (DIRECT) {
    if (first) direct_tile<MODE_DW, 2, 2, T / 2, T / 2, 64, 2, false>(pw, block, blocks);
    else direct_tile<MODE_DX, 2, 2, T / 2, T / 2, 64, 2, false>(px, block, blocks);
  } else {
    if (first) any_tile<MODE_DW, T, T, false>(pw, block, blocks);
    else any_tile<MODE_DX, T, T, false>(px, block, blocks);
  }
}

// ------------------------------------------------------------------------------------------------ fp32 (parity mode)
// four consecutive elements of which n >= 1 exist (the others are zero)
DEVINL f32x4 load4(const float* p, int n) {
  if (n >= 4) return *(const f32x4_any*)p;
  const float a = p[0], b = p[min(1, n - 1)], c = p[min(2, n - 1)];
  return f32x4{a, n > 1 ? b : 0.f, n > 2 ? c : 0.f, 0.f};
}

// One operand tile, as Tile: T rows x 32 contraction elements, 256 threads, 16-byte granules through registers.
// KC image [T][32 + 4]: a lane's fragment is the four consecutive k of one 16-byte read, rows 36 floats apart on banks of their own.
// RC image [32][T + 4]: four 4-byte reads, k rows 4 apart 16 banks apart.
// WHOLE: no granule is cut by the end of its row (ragged ones are fetched as the row's last four elements and shifted).
// Either way MFMA e of a group of four takes element e of both operands: the sum runs over all k, in whatever order.
constexpr int FK = 32;
template <bool RC, int T, bool WHOLE> struct F32Tile {
  static constexpr int NG = T * FK / 4 / 256, PITCH = RC ? T + 4 : FK + 4, FLOATS = (RC ? FK : T) * PITCH, TG = T / 4, KG = FK / 4;
  const float* src[NG];
  int kof[NG], len[NG], cut[NG];
  f32x4 v[NG];
  bool few;

  DEVINL void init(const float* base, int ld, int row0, int rows, int kbeg, int clen) {
    few = (RC ? rows : clen) < 4;
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      const int idx = threadIdx.x + u * 256;
      const int r = row0 + (RC ? idx % TG * 4 : idx / KG);
      kof[u] = RC ? idx / TG : idx % KG * 4;
      len[u] = rows - r;
      src[u] = r >= rows ? nullptr : RC ? base + (size_t)(kbeg + kof[u]) * ld + r : base + (size_t)r * ld + kbeg + kof[u];
    }
  }
  DEVINL void request(size_t k, int ld, int left) {
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      const bool ok = src[u] != nullptr && kof[u] < left;
      const float* q = src[u] + (RC ? k * ld : k);
      if (WHOLE) {
        v[u] = *(ok ? (const f32x4_any*)q : (const f32x4_any*)&zero_granule);
        continue;
      }
      const int n = RC ? len[u] : left - kof[u];
      cut[u] = ok && n < 4 && !few ? 4 - n : 0;
      if (few) v[u] = ok ? load4(q, n) : f32x4{0.f, 0.f, 0.f, 0.f};
      else v[u] = *(ok ? (const f32x4_any*)(q - cut[u]) : (const f32x4_any*)&zero_granule);
    }
  }
  DEVINL void commit(float* img) {
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      const int idx = threadIdx.x + u * 256;
      f32x4 t = v[u];
      if (WHOLE) cut[u] = 0;
      if (cut[u] == 1) t = f32x4{t[1], t[2], t[3], 0.f};
      if (cut[u] == 2) t = f32x4{t[2], t[3], 0.f, 0.f};
      if (cut[u] == 3) t = f32x4{t[3], 0.f, 0.f, 0.f};
      *(f32x4*)(img + (RC ? idx / TG * PITCH + idx % TG * 4 : idx / KG * PITCH + idx % KG * 4)) = t;
    }
  }
  // 16 rows from r0, contraction elements 16 kk .. 16 kk + 15
  static DEVINL f32x4 frag(const float* img, int r0, int kk) {
    const int lane = threadIdx.x & 63, k = kk * 16 + 4 * (lane >> 4), r = r0 + (lane & 15);
    if (!RC) return *(const f32x4*)(img + r * PITCH + k);
    f32x4 f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = img[(k + e) * PITCH + r];
    return f;
  }
};

template <int MODE> DEVINL void f32_store(const LinP& p, int slab, int i, int j, f32x4 v) {
  const int n = p.J - j;
  if (i >= p.I || n <= 0) return;
  float* o = MODE == MODE_DW ? (float*)p.out + ((size_t)slab * p.I + i) * p.J + j : (float*)p.out + (size_t)i * p.o_ld + j;
  const float* r = MODE == MODE_FWD ? (p.res ? (const float*)p.res + (size_t)i * p.r_ld + j : nullptr) : MODE == MODE_DX && p.accumulate ? o : nullptr;
  f32x4 add = {0.f, 0.f, 0.f, 0.f};
  if (r) add = load4(r, n);
  if (MODE == MODE_FWD) {
    if (p.bias) v += load4(p.bias + j, n);
    if (p.z) {
      float* z = (float*)p.z + (size_t)i * p.z_ld + j;
      if (n >= 4) *(f32x4_any*)z = v;
      else
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (e < n) z[e] = v[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = act_fwd_precise(v[e], p.act);
  }
  if (r) v += add;
  if (n >= 4) *(f32x4_any*)o = v;
  else
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < n) o[e] = v[e];
}

// T x T tile, four waves of T / 2 x T / 2, v_mfma_f32_16x16x4_f32, two LDS images per operand, one barrier per stage, whole operands two stages
// ahead (12800 x 512 x 512 82 us, 82 TFLOP/s; one ahead 103)
template <int MODE, int T, bool WHOLE> __global__ __launch_bounds__(256) void linear_f32_kernel(const LinP p) {
  typedef F32Tile<MODE == MODE_DW, T, WHOLE> TA;
  typedef F32Tile<MODE != MODE_FWD, T, WHOLE> TB;
  constexpr int F = T / 32, STAGE = TA::FLOATS + TB::FLOATS, AHEAD = WHOLE ? 2 : 1;
  extern __shared__ __align__(16) float fsmem[];
  const Place at = place<T, T>(p, blockIdx.x, gridDim.x);
  const int i0 = at.i0, j0 = at.j0;
  const int wave = threadIdx.x >> 6, wi = (wave >> 1) * (T / 2), wj = (wave & 1) * (T / 2), lane = threadIdx.x & 63;
  const int kbeg = at.slab * p.ksteps * FK;
  const int klen = (MODE == MODE_DW ? min(p.Kc, kbeg + p.ksteps * FK) : p.Kc) - kbeg;
  f32x4 acc[F][F];
#pragma unroll
  for (int a = 0; a < F; ++a)
#pragma unroll
    for (int b = 0; b < F; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  TA ta[AHEAD];
  TB tb[AHEAD];
#pragma unroll
  for (int h = 0; h < AHEAD; ++h) {
    ta[h].init((const float*)p.a, p.a_ld, i0, p.I, kbeg, p.Kc);
    tb[h].init((const float*)p.b, p.b_ld, j0, p.J, kbeg, p.Kc);
    ta[h].request(h * FK, p.a_ld, klen - h * FK);
    tb[h].request(h * FK, p.b_ld, klen - h * FK);
  }
  for (int k = 0; k < klen; k += 2 * FK) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k0 = k + h * FK, next = k0 + AHEAD * FK;
      if (k0 >= klen) break;
      float *ia = fsmem + h * STAGE, *ib = ia + TA::FLOATS;
      ta[h % AHEAD].commit(ia);
      tb[h % AHEAD].commit(ib);
      __syncthreads();      // image h is whole; image h ^ 1 was last read before every wave came here
      ta[h % AHEAD].request(next, p.a_ld, klen - next);      // (past the end: zeros; a branch here would make every wait one for all loads)
      tb[h % AHEAD].request(next, p.b_ld, klen - next);
#pragma unroll
      for (int kk = 0; kk < FK / 16; ++kk) {
        f32x4 fa[F], fb[F];
#pragma unroll
        for (int a = 0; a < F; ++a) fa[a] = TA::frag(ia, wi + a * 16, kk);
#pragma unroll
        for (int b = 0; b < F; ++b) fb[b] = TB::frag(ib, wj + b * 16, kk);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int a = 0; a < F; ++a)
#pragma unroll
            for (int b = 0; b < F; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[b][e], fa[a][e], acc[a][b], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int a = 0; a < F; ++a)
#pragma unroll
    for (int b = 0; b < F; ++b) f32_store<MODE>(p, at.slab, i0 + wi + a * 16 + (lane & 15), j0 + wj + b * 16 + 4 * (lane >> 4), acc[a][b]);
}

// Few output values (forward only: both operands run along the contraction, so fragments come straight from memory): one workgroup per block of
// 16 R x 16 R values, the contraction split over its waves with every load of a step in flight at once, partial blocks added in wave order.
// Rows beyond the last are clamped to it; what they give is not stored.  fp32: a lane's four consecutive k feed four MFMAs in turn.
DEVINL u32x4 load_granule(const bf16_t* p, int n) { return load8(p, n); }
DEVINL u32x4 load_granule(const float* p, int n) {
  const f32x4 v = load4(p, n);
  return *(const u32x4*)&v;
}
DEVINL f32x4 granule_mma(const bf16_t*, const u32x4& a, const u32x4& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8*)&b, *(const bf16x8*)&a, c, 0, 0, 0);
}
DEVINL f32x4 granule_mma(const float*, const u32x4& a, const u32x4& b, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b[e]), __uint_as_float(a[e]), c, 0, 0, 0);
  return c;
}
template <typename T, int R, bool HEAVY> __global__ __launch_bounds__(1024) void linear_blocks_kernel(const LinP p, const int kper) {
  constexpr int E = 16 / (int)sizeof(T), STEP = 4 * E, U = sizeof(T) == 4 && R == 2 ? 2 : 4;      // (four would spill)
  extern __shared__ f32x4 part[];       // [waves][R * R][64]
  const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int i0 = (int)(blockIdx.x / p.nj) * (16 * R), j0 = (int)(blockIdx.x % p.nj) * (16 * R), ko = E * (lane >> 4);
  const T *pa[R], *pb[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    pa[r] = (const T*)p.a + (size_t)min(i0 + r * 16 + (lane & 15), p.I - 1) * p.a_ld + ko;
    pb[r] = (const T*)p.b + (size_t)min(j0 + r * 16 + (lane & 15), p.J - 1) * p.b_ld + ko;
  }
  const int k0 = wave * kper, k1 = min(p.Kc, k0 + kper);
  f32x4 acc[R][R];
#pragma unroll
  for (int a = 0; a < R; ++a)
#pragma unroll
    for (int b = 0; b < R; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k = k0; k < k1; k += U * STEP) {
    u32x4 fa[U][R], fb[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = k + u * STEP, n = k1 - at - ko;
      if (at + STEP <= k1) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          fa[u][r] = *(const u32x4_any*)(pa[r] + at);
          fb[u][r] = *(const u32x4_any*)(pb[r] + at);
        }
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          fa[u][r] = n > 0 ? load_granule(pa[r] + at, n) : u32x4{0u, 0u, 0u, 0u};
          fb[u][r] = n > 0 ? load_granule(pb[r] + at, n) : u32x4{0u, 0u, 0u, 0u};
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int a = 0; a < R; ++a)
#pragma unroll
        for (int b = 0; b < R; ++b) acc[a][b] = granule_mma((const T*)nullptr, fa[u][a], fb[u][b], acc[a][b]);
  }
  auto store = [&](int f, f32x4 v) {
    const int i = i0 + f / R * 16 + (lane & 15), j = j0 + f % R * 16 + 4 * (lane >> 4);
    if constexpr (sizeof(T) == 2) store4<HEAVY>(p, i, j, v, bias4<MODE_FWD>(p, j));
    else f32_store<MODE_FWD>(p, 0, i, j, v);
  };
  if (waves == 1) {
#pragma unroll
    for (int f = 0; f < R * R; ++f) store(f, acc[f / R][f % R]);
    return;
  }
#pragma unroll
  for (int f = 0; f < R * R; ++f) part[(wave * R * R + f) * 64 + lane] = acc[f / R][f % R];
  __syncthreads();
  for (int f = wave; f < R * R; f += waves) {
    f32x4 v = part[f * 64 + lane];
    for (int w = 1; w < waves; ++w) v += part[(w * R * R + f) * 64 + lane];
    store(f, v);
  }
}

// ------------------------------------------------------------------------------------------------ dz, db, slab sums
DEVINL void load_vec(const bf16_t* p, int n, float (&f)[8]) { Vec<bf16_t>::cvt(load8(p, n), f); }
DEVINL void load_vec(const float* p, int n, float (&f)[4]) { Vec<float>::cvt(load4(p, n), f); }
template <bool PRECISE> DEVINL float dz_act_grad(float u, int act) {
  if (!PRECISE && act == PLYOLO_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(u * -1.4426950408889634f));
    return fmaf(s, fmaf(-u, s, u), s);
  }
  return act_grad<PRECISE>(u, act);
}

struct DzP {
  const void* dy;
  const void* z;        // NULL: dz = dy (only the column sums are formed)
  void* dz;             // [M][dz_ld], columns N .. dz_ld zero; NULL with z
  float* part;          // [blocks][N] column sums, or NULL
  int M, N, dy_ld, z_ld, dz_ld, act, rows;
};

// dz and the column sums of `rows` rows: a thread owns one vector of columns (16 bytes of T, at any element address) and walks down the rows.
// dz leaves with a pitch of whole vectors and zeros behind column N: the products then take it on their wide path whatever N is.
// HBM: 51200 x 256 bf16 21 us, 3.7 TB/s (the kernel alone; cached 18).
template <typename T> __global__ __launch_bounds__(256) void linear_dz_kernel(const DzP p) {
  constexpr int V = Vec<T>::N, U = 4;
  __shared__ float red[256 * V];
  const int cv = (p.N + V - 1) / V, cols = min(cv, 256), rpb = 256 / cols;
  const int tcol = threadIdx.x % cols, trow = threadIdx.x / cols;
  const int64_t m0 = (int64_t)blockIdx.x * p.rows;
  const int nr = (int)min((int64_t)p.rows, (int64_t)p.M - m0);
  for (int cb = 0; cb < cv; cb += cols) {
    const int col = cb + tcol, n = p.N - col * V;        // n < V: the last, partial vector
    float s[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = 0.f;
    if (col < cv && trow < rpb) {
      const T* pd = (const T*)p.dy + (size_t)m0 * p.dy_ld + col * V;
      const T* pz = p.z ? (const T*)p.z + (size_t)m0 * p.z_ld + col * V : nullptr;
      T* po = p.dz ? (T*)p.dz + (size_t)m0 * p.dz_ld + col * V : nullptr;
      for (int r0 = trow; r0 < nr; r0 += U * rpb) {
        float d[U][V], z[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (r0 + u * rpb < nr) {
            load_vec(pd + (size_t)(r0 + u * rpb) * p.dy_ld, n, d[u]);
            if (pz) load_vec(pz + (size_t)(r0 + u * rpb) * p.z_ld, n, z[u]);
          }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (r0 + u * rpb < nr) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              if (pz) d[u][e] *= dz_act_grad<Vec<T>::precise>(z[u][e], p.act);
              s[e] += d[u][e];
            }
            if (po) Vec<T>::store(po + (size_t)(r0 + u * rpb) * p.dz_ld, d[u]);
          }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) red[(trow * cols + tcol) * V + e] = s[e];
    }
    if (p.part) {
      __syncthreads();
      const int nch = min(cols, cv - cb) * V;
      for (int t = threadIdx.x; t < nch; t += 256)
        if (cb * V + t < p.N) {
          float a = 0.f;
          for (int w = 0; w < rpb && w < nr; ++w) a += red[w * cols * V + t];
          p.part[(size_t)blockIdx.x * p.N + cb * V + t] = a;
        }
      __syncthreads();
    }
  }
}

// out[e] (+)= sum over S slabs of part[s][e] in a fixed order: 4 E elements x 64 / E slab lanes per workgroup, eight slabs in flight per lane.
// The weight gradient's workgroups (E by its slab count) come first, the bias gradient's (E = 4) behind them: one launch for both.
struct FoldP {
  const float* part;
  void* out;
  size_t elems;
  int S, f32, blocks;
};
template <int E> DEVINL void fold(const FoldP& q, int block, int accumulate, f32x4* red) {
  constexpr int L = 256 / E;
  const size_t e = ((size_t)block * E + threadIdx.x % E) * 4;
  const int sl = threadIdx.x / E, n = q.elems > e ? (q.elems - e < 4 ? (int)(q.elems - e) : 4) : 0;
  const bool whole = q.elems % 4 == 0;       // (every slab then starts on a 16-byte boundary)
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (n > 0) {
#pragma unroll 8
    for (int s = sl; s < q.S; s += L) {
      const float* r = q.part + (size_t)s * q.elems + e;
      if (whole) v += *(const f32x4*)r;
      else v += load4(r, n);
    }
  }
  red[threadIdx.x] = v;
  __syncthreads();
  for (int h = L / 2; h > 0; h >>= 1) {
    if (sl < h) red[threadIdx.x] += red[threadIdx.x + h * E];
    __syncthreads();
  }
  if (sl == 0) {
    v = red[threadIdx.x];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) {
        if (q.f32) {
          float* o = (float*)q.out + e + k;
          *o = accumulate ? *o + v[k] : v[k];
        } else {
          bf16_t* o = (bf16_t*)q.out + e + k;
          *o = f2bf(accumulate ? bf2f(*o) + v[k] : v[k]);
        }
      }
  }
}
// 4 * fold_width elements per workgroup: by slab count, so that the lanes of an element have up to eight slabs each
// (3 slabs of 1024 x 1024 by sixteen lanes 13 us, by one 5)
__host__ __device__ __forceinline__ int fold_width(int slabs) { return slabs <= 8 ? 256 : slabs <= 32 ? 64 : slabs <= 64 ? 16 : 4; }
__global__ __launch_bounds__(256) void linear_fold_kernel(const FoldP w, const FoldP b, const int accumulate) {
  __shared__ f32x4 red[256];
  if ((int)blockIdx.x >= w.blocks) fold<4>(b, blockIdx.x - w.blocks, accumulate, red);
  else if (fold_width(w.S) == 4) fold<4>(w, blockIdx.x, accumulate, red);
  else if (fold_width(w.S) == 16) fold<16>(w, blockIdx.x, accumulate, red);
  else if (fold_width(w.S) == 64) fold<64>(w, blockIdx.x, accumulate, red);
  else fold<256>(w, blockIdx.x, accumulate, red);
}

// ------------------------------------------------------------------------------------------------ host side
struct BwdPlan {
  int dz_ld, S, ksteps, dzblk, dzrows, tile;
  size_t dz_bytes, part_off, part_bytes, slab_off, slab_bytes, total;
};

size_t up16(size_t v) { return (v + 15) & ~(size_t)15; }

// Tile of an I x J output: the larger, the fewer LDS reads per MFMA and the fewer re-reads of the operands; the smaller, the more of the chip a
// small output fills.  256 (x 256, eight waves: one workgroup per compute unit) becomes 224 x 256 where that is still one round of the 256
// compute units: 12800 x 2048 x 1024 67 -> 64 us, 12800 x 1024 x 1024 40 -> 38 us.  128 x 128 in place of 256 x 256: 82 and 47 us.
// fp32 and operands that pass registers (direct false): 128 or 64.
int pick_tile(int64_t I, int64_t J, int64_t Kc, bool direct) {
  auto tiles = [&](int a, int b) { return ((I + a - 1) / a) * ((J + b - 1) / b); };
  if (direct && tiles(256, 256) >= 128 && J > 128 && Kc >= 512) return tiles(224, 256) <= 256 ? 224 : 256;
  if (tiles(128, 128) >= 192 && J > 64) return 128;
  return 64;
}

// Tile and slabs of dw: enough row ranges to give every compute unit a workgroup, as long as the slabs are not more to move than the operands; a
// layer that does not get there with 128 x 128 tiles takes small ones, and so does one whose output fills half of them (K <= 64, where dx has
// small tiles too and the two share a launch: 204800 x 64 x 64 bf16 66 -> 52 us; fp32, N <= 64 also: 204800 x 128 x 64 171 -> 151).
// bf16: three quarters of the compute units where dx shares the launch (backward, three quarters / all / one and a half: 51200 x 256 x 256
// 59.9 / 59.9 / 67 us, 204800 x 128 x 128 85.6 / 86.8 / 89.5, 25600 x 512 x 256 49 / 51 / 53), two workgroups each where dx has its own large
// tiles (two / three quarters / three: 12800 x 2048 x 1024 182 / 234 / 200, 12800 x 1024 x 1024 115 / 157 / 127, 25600 x 1024 x 512
// 118 / 160 / 136).
void dw_plan(const plyolo_linear_desc* d, int tile, BwdPlan* b) {
  const bool half = d->dtype == PLYOLO_BF16;
  const int64_t tiles = (int64_t)cdiv(d->N, tile) * cdiv(d->K, tile);
  const int steps = cdiv(d->M, half ? BK : FK);
  const double slab = 4.0 * d->N * d->K, operands = (half ? 2.0 : 4.0) * d->M * ((double)d->N + d->K);
  const int want = !half ? 256 : pick_tile(d->M, d->K, d->N, true) > 128 ? 512 : 192;
  int64_t s = (want + tiles - 1) / tiles;
  if (s > operands / slab) s = (int64_t)(operands / slab);
  if (s > steps) s = steps;
  if (s < 1) s = 1;
  b->tile = tile;
  b->ksteps = (int)((steps + s - 1) / s);
  b->S = (steps + b->ksteps - 1) / b->ksteps;
}

BwdPlan bwd_plan(const plyolo_linear_desc* d) {
  BwdPlan b{};
  const bool half = d->dtype == PLYOLO_BF16;
  const int es = half ? 2 : 4;
  b.dz_ld = (d->N + 7) & ~7;
  b.dz_bytes = d->act == PLYOLO_ACT_NONE ? 0 : up16((size_t)d->M * b.dz_ld * es);
  // one row a thread, 4 to 16 (400 x 333 x 777 backward 35 us with 16 rows whatever N, 26 with 4), and at most 1024 workgroups
  b.dzrows = max(min(max(4, 256 / min(cdiv(d->N, half ? 8 : 4), 256)), 16), cdiv(d->M, 1024));
  b.dzblk = cdiv(d->M, b.dzrows);
  b.part_off = b.dz_bytes;
  b.part_bytes = up16((size_t)b.dzblk * d->N * 4);
  b.slab_off = b.part_off + b.part_bytes;
  dw_plan(d, 128, &b);
  const bool thin = d->K <= 64 || (!half && d->N <= 64);
  if (thin || (int64_t)b.S * cdiv(d->N, 128) * cdiv(d->K, 128) < 128) dw_plan(d, 64, &b);
  b.slab_bytes = up16((size_t)b.S * d->N * d->K * 4);
  b.total = b.slab_off + b.slab_bytes;
  return b;
}

int check_linear(const plyolo_linear_desc* d, const char* who) {
  PLY_CHECK_ARG(d != nullptr, "%s: null descriptor", who);
  PLY_CHECK_ARG(d->dtype == PLYOLO_BF16 || d->dtype == PLYOLO_F32, "%s: bad dtype %d", who, d->dtype);
  PLY_CHECK_ARG(d->M > 0 && d->N > 0 && d->K > 0, "%s: non-positive dimension (M %d, N %d, K %d)", who, d->M, d->N, d->K);
  PLY_CHECK_ARG(d->N <= (1 << 20) && d->K <= (1 << 20) && (double)d->N * d->K < 1073741824.0 && d->M <= 2147483647 - 1024, "%s: dimension too large (M %d, N %d, K %d)", who, d->M, d->N, d->K);
  PLY_CHECK_ARG(d->act >= PLYOLO_ACT_NONE && d->act <= PLYOLO_ACT_GELU, "%s: bad activation %d", who, d->act);
  PLY_CHECK_ARG(d->x_ld >= d->K && d->w_ld >= d->K, "%s: x_ld %d or w_ld %d < K %d", who, d->x_ld, d->w_ld, d->K);
  return 0;
}

// workgroups of an I x J output (a launch has fewer than 2^32 threads: those of up to 512, two such grids in one launch, 64 for the many small ones)
int tile_grid(LinP& p, int tile, int slabs, const char* who) {
  p.nj = cdiv(p.J, tile == 224 ? 256 : tile);
  const int64_t n = (int64_t)cdiv(p.I, tile) * p.nj;
  PLY_CHECK_ARG(n * slabs < (tile < 64 ? 67108864 : 8388608), "%s: more than %d workgroups", who, tile < 64 ? 67108864 : 8388608);
  p.tiles = (int)n;
  return (int)n * slabs;
}

bool rows16(const void* p, int ld, int len) { return (size_t)p % 16 == 0 && ld % 8 == 0 && len % 8 == 0; }

template <int MODE, int TI, int TJ> size_t tile_lds(size_t stages) {
  const size_t out = MODE == MODE_DW ? 0 : out_bytes<TI, TJ>();
  return out > stages ? out : stages;
}
template <int MODE, int T, bool HEAVY> hipError_t launch_any(const LinP& p, int grid, hipStream_t s) {
  const size_t lds = tile_lds<MODE, T, T>(2 * (size_t)(2 * T) * BK * 2);
  auto k = linear_bf16_any_kernel<MODE, T, HEAVY>;
  if (hipError_t e = plyolo::ensure_dynamic_lds((const void*)k, lds); e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3(grid), dim3(256), lds, s, p);
  return hipGetLastError();
}
template <int MODE, int NWI, int NWJ, int WI, int WJ, int K, int ST, bool HEAVY> hipError_t launch_direct(const LinP& p, int grid, hipStream_t s) {
  constexpr int TI = NWI * WI, TJ = NWJ * WJ;
  const size_t lds = tile_lds<MODE, TI, TJ>(ST * (size_t)(TI + TJ) * K * 2);
  auto k = linear_bf16_kernel<MODE, NWI, NWJ, WI, WJ, K, ST, HEAVY>;
  if (hipError_t e = plyolo::ensure_dynamic_lds((const void*)k, lds); e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3(grid), dim3(64 * NWI * NWJ), lds, s, p);
  return hipGetLastError();
}
template <typename T, int R, bool HEAVY> hipError_t launch_blocks_of(const LinP& p, int grid, int waves, int kper, hipStream_t s) {
  const size_t lds = waves > 1 ? (size_t)waves * R * R * 64 * sizeof(f32x4) : 0;
  auto k = linear_blocks_kernel<T, R, HEAVY>;
  hipLaunchKernelGGL(k, dim3(grid), dim3(64 * waves), lds, s, p, kper);
  return hipGetLastError();
}
template <typename T, bool HEAVY> hipError_t launch_blocks(int R, const LinP& p, int grid, int waves, int kper, hipStream_t s) {
  return R == 1 ? launch_blocks_of<T, 1, HEAVY>(p, grid, waves, kper, s)
                : launch_blocks_of<T, 2, HEAVY>(p, grid, waves, kper, s);
}
template <int MODE, int T, bool WHOLE> hipError_t launch_f32(const LinP& p, int grid, hipStream_t s) {
  constexpr size_t lds = 2 * (size_t)(F32Tile<MODE == MODE_DW, T, WHOLE>::FLOATS + F32Tile<MODE != MODE_FWD, T, WHOLE>::FLOATS) * sizeof(float);
  auto k = linear_f32_kernel<MODE, T, WHOLE>;
  if (hipError_t e = plyolo::ensure_dynamic_lds((const void*)k, lds); e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3(grid), dim3(256), lds, s, p);
  return hipGetLastError();
}
// direct: both operands' granules are whole and 16-byte aligned
template <int MODE, bool HEAVY> hipError_t launch_bf16(const LinP& p, int tile, int grid, bool direct, hipStream_t s) {
  if (direct) {
    if constexpr (MODE != MODE_DW) {
      if (tile == 256) return launch_direct<MODE, 2, 4, 128, 64, 64, 2, HEAVY>(p, grid, s);
      if (tile == 224) return launch_direct<MODE, 2, 4, 112, 64, 64, 2, HEAVY>(p, grid, s);
    }
    if (tile == 128) return launch_direct<MODE, 2, 2, 64, 64, 64, 2, HEAVY>(p, grid, s);
    return launch_direct<MODE, 2, 2, 32, 32, 64, 3, HEAVY>(p, grid, s);
  }
  return tile == 128 ? launch_any<MODE, 128, HEAVY>(p, grid, s) : launch_any<MODE, 64, HEAVY>(p, grid, s);
}
template <int T, bool DIRECT> hipError_t launch_both(const LinP& px, const LinP& pw, int gx, int gw, hipStream_t s) {
  const size_t lds = tile_lds<MODE_DX, T, T>(2 * (size_t)(2 * T) * 64 * 2);
  auto k = linear_bf16_bwd_kernel<T, DIRECT>;
  if (hipError_t e = plyolo::ensure_dynamic_lds((const void*)k, lds); e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3((unsigned)gx + (unsigned)gw), dim3(256), lds, s, px, pw, gw);
  return hipGetLastError();
}
template <int MODE> hipError_t launch_gemm(int dtype, const LinP& p, int tile, int grid, bool direct, hipStream_t s) {
  if (dtype != PLYOLO_BF16) {
    const bool whole = (MODE == MODE_DW ? p.I % 4 : p.Kc % 4) == 0 && (MODE == MODE_FWD ? p.Kc % 4 : p.J % 4) == 0;
    if (whole) return tile == 128 ? launch_f32<MODE, 128, true>(p, grid, s) : launch_f32<MODE, 64, true>(p, grid, s);
    return tile == 128 ? launch_f32<MODE, 128, false>(p, grid, s) : launch_f32<MODE, 64, false>(p, grid, s);
  }
  if (MODE == MODE_FWD && p.act > PLYOLO_ACT_LRELU) return launch_bf16<MODE, MODE == MODE_FWD>(p, tile, grid, direct, s);
  return launch_bf16<MODE, false>(p, tile, grid, direct, s);
}

}  // namespace

extern "C" {

size_t plyolo_linear_workspace(const plyolo_linear_desc* d, int backward) {
  if (check_linear(d, "linear_workspace")) return 0;
  return backward ? bwd_plan(d).total : 0;
}

int plyolo_linear_fwd(const plyolo_linear_desc* d, const void* x, const void* w, const float* bias, const void* res, void* z, void* y,
                      void* workspace, size_t ws_bytes, void* stream) {
  if (check_linear(d, "linear_fwd")) return -1;
  PLY_CHECK_ARG(x && w && y, "linear_fwd: null operand");
  PLY_CHECK_ARG(d->y_ld >= d->N && (!z || d->z_ld >= d->N) && (!res || d->r_ld >= d->N), "linear_fwd: a row pitch is smaller than N = %d", d->N);
  const size_t es = d->dtype == PLYOLO_BF16 ? 2 : 4;
  PLY_CHECK_ARG(((size_t)x | (size_t)w | (size_t)res | (size_t)z | (size_t)y) % es == 0 && (size_t)bias % 4 == 0, "linear_fwd: misaligned operand");
  LinP p{};
  p.a = x; p.b = w; p.out = y; p.z = z; p.res = res; p.bias = bias;
  p.I = d->M; p.J = d->N; p.Kc = d->K;
  p.a_ld = d->x_ld; p.b_ld = d->w_ld; p.o_ld = d->y_ld; p.z_ld = d->z_ld; p.r_ld = d->r_ld;
  p.act = d->act;
  p.vec4 = d->y_ld % 4 == 0 && (!z || d->z_ld % 4 == 0) && (!res || d->r_ld % 4 == 0) && ((size_t)y | (size_t)z | (size_t)res) % 8 == 0;
  const int dtype = d->dtype;
  const double m = d->M, n = d->N, k = d->K;
  plyolo::annotate("linear_fwd", 2.0 * m * n * k, (m * k + n * k + m * n * (1.0 + (z ? 1 : 0) + (res ? 1 : 0))) * es);
  // Blocks of 16 R x 16 R re-read x once per 16 R columns and w once per 16 R rows, out of L2; a tile walks its whole contraction by itself.
  // Estimated microseconds, fitted over M 16 .. 51200, N 16 .. 2048, K 32 .. 2048.  Measured, M x K x N, us with R = 1 / R = 2 / tiles:
  //   bf16  64 x 2048 x 1024  6.6 / 10.4 / 13.6   256 x 1024 x 1024  10.2 /  7.2 /  9.0   12800 x 64 x 64  6.5 / 5.1 / 4.4
  //   fp32  64 x 2048 x 1024 10.7 / 22.2 / 53.3   256 x 1024 x 1024  18.5 / 13.8 / 30.8   3200 x 512 x 512  54 / 37 / 27.0
  const bool half = dtype == PLYOLO_BF16;
  auto again = [&](int e) { return (m * k * cdiv(d->N, e) + n * k * cdiv(d->M, e)) * es; };
  const double one_us = half ? 3.4 + again(16) / 9.6e6 : 6.0 + again(16) / 9.0e6, two_us = half ? 3.6 + again(32) / 8.0e6 : 5.0 + again(32) / 7.5e6;
  const double tiles_us = half ? 4.0 + k * 0.31 / 64 : 6.5 + k / (d->K % 4 == 0 ? 43 : 29);
  const bool fill = (int64_t)cdiv(d->M, 32) * cdiv(d->N, 32) >= 192;      // blocks of 32 leave too many of the 256 CUs without work below this
  const int R = fill && two_us < one_us ? 2 : 1;
  if ((R == 2 ? two_us : one_us) < tiles_us) {
    const int grid = tile_grid(p, 16 * R, 1, "linear_fwd");
    if (grid < 0) return -1;
    const int step = half ? 32 : 16;
    int waves = 1;
    while (waves < 16 && waves * 2 * step <= d->K && (int64_t)grid * waves < 4096) waves *= 2;
    const int kper = cdiv(cdiv(d->K, waves), step) * step;
    return plyolo::submit(stream, [=](hipStream_t s) -> hipError_t {
      return !half                       ? launch_blocks<float, false>(R, p, grid, waves, kper, s)
             : p.act > PLYOLO_ACT_LRELU ? launch_blocks<bf16_t, true>(R, p, grid, waves, kper, s)
                                        : launch_blocks<bf16_t, false>(R, p, grid, waves, kper, s);
    });
  }
  const bool direct = rows16(x, d->x_ld, d->K) && rows16(w, d->w_ld, d->K);
  const int tile = pick_tile(d->M, d->N, d->K, direct && dtype == PLYOLO_BF16);
  const int grid = tile_grid(p, tile, 1, "linear_fwd");
  if (grid < 0) return -1;
  return plyolo::submit(stream, [=](hipStream_t s) -> hipError_t { return launch_gemm<MODE_FWD>(dtype, p, tile, grid, direct, s); });
}

int plyolo_linear_bwd(const plyolo_linear_desc* d, const void* dy, const void* z, const void* x, const void* w, void* dx, int dx_ld,
                      int accumulate_dx, void* dw, int dw_dtype, float* db, int accumulate_params, void* workspace, size_t ws_bytes, void* stream) {
  if (check_linear(d, "linear_bwd")) return -1;
  PLY_CHECK_ARG(dy && (z || d->act == PLYOLO_ACT_NONE), "linear_bwd: null dy, or null z with an activation");
  PLY_CHECK_ARG(dx || dw || db, "linear_bwd: nothing to compute");
  PLY_CHECK_ARG((!dx || w) && (!dw || x), "linear_bwd: dx needs w, dw needs x");
  PLY_CHECK_ARG(d->y_ld >= d->N && (!z || d->z_ld >= d->N) && (!dx || dx_ld >= d->K), "linear_bwd: a row pitch is smaller than its row (y_ld %d, z_ld %d, dx_ld %d)", d->y_ld, d->z_ld, dx_ld);
  PLY_CHECK_ARG(!dw || dw_dtype == PLYOLO_F32 || dw_dtype == d->dtype, "linear_bwd: dw_dtype must be PLYOLO_F32 or the descriptor's dtype");
  const size_t es = d->dtype == PLYOLO_BF16 ? 2 : 4;
  PLY_CHECK_ARG(((size_t)dy | (size_t)z | (size_t)x | (size_t)w | (size_t)dx) % es == 0 && (size_t)dw % (dw_dtype == PLYOLO_F32 ? 4 : 2) == 0 && (size_t)db % 4 == 0,
                "linear_bwd: misaligned operand");
  const BwdPlan b = bwd_plan(d);
  PLY_CHECK_ARG(workspace && (size_t)workspace % 16 == 0 && ws_bytes >= b.total, "linear_bwd: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", b.total, ws_bytes);
  unsigned char* ws = (unsigned char*)workspace;
  const int dtype = d->dtype;
  const bool has_act = d->act != PLYOLO_ACT_NONE;
  DzP q{};
  q.dy = dy; q.M = d->M; q.N = d->N; q.dy_ld = d->y_ld; q.z_ld = d->z_ld; q.act = d->act; q.rows = b.dzrows;
  q.z = has_act ? z : nullptr;
  q.dz = has_act && (dx || dw) ? ws : nullptr;
  q.dz_ld = b.dz_ld;
  q.part = db ? (float*)(ws + b.part_off) : nullptr;
  LinP px{}, pw{};
  const void* g = has_act ? (const void*)ws : dy;
  const int g_ld = has_act ? b.dz_ld : d->y_ld;
  px.a = g; px.b = w; px.out = dx; px.I = d->M; px.J = d->K;
  px.Kc = d->N;
  px.a_ld = g_ld; px.b_ld = d->w_ld; px.o_ld = dx_ld; px.accumulate = accumulate_dx ? 1 : 0;
  pw.a = g; pw.b = x; pw.out = ws + b.slab_off; pw.I = d->N; pw.J = d->K; pw.Kc = d->M;
  pw.a_ld = g_ld; pw.b_ld = d->x_ld; pw.ksteps = b.ksteps;
  pw.vec4 = d->K % 4 == 0;
  // dz rows are padded to whole vectors of zeros, dy rows end at N
  const int g_len = has_act ? b.dz_ld : d->N;
  const bool dx_direct = rows16(g, g_ld, g_len) && rows16(w, d->w_ld, d->K), dw_direct = rows16(g, g_ld, g_len) && rows16(x, d->x_ld, d->K);
  const int tx = pick_tile(d->M, d->K, d->N, dx_direct && dtype == PLYOLO_BF16);
  const int gx = tile_grid(px, tx, 1, "linear_bwd"), gw = tile_grid(pw, b.tile, b.S, "linear_bwd");
  if (gx < 0 || gw < 0) return -1;
  FoldP fw{}, fb{};
  if (dw) {
    fw.part = (const float*)(ws + b.slab_off); fw.out = dw; fw.elems = (size_t)d->N * d->K; fw.S = b.S; fw.f32 = dw_dtype == PLYOLO_F32;
    fw.blocks = (int)cdivz(fw.elems, 4 * fold_width(fw.S));
  }
  if (db) {
    fb.part = q.part; fb.out = db; fb.elems = (size_t)d->N; fb.S = b.dzblk; fb.f32 = 1;
    fb.blocks = (int)cdivz(fb.elems, 16);
  }
  const int acc = accumulate_params ? 1 : 0;
  const double m = d->M, n = d->N, k = d->K;
  plyolo::annotate("linear_bwd", 2.0 * m * n * k * ((dx ? 1 : 0) + (dw ? 1 : 0)), (m * n * (has_act ? 2.0 : 1.0) + 2.0 * m * k + 2.0 * n * k) * es);
  return plyolo::submit(stream, [=](hipStream_t s) -> hipError_t {
    if (q.dz || q.part) {
      if (dtype == PLYOLO_BF16) hipLaunchKernelGGL(linear_dz_kernel<bf16_t>, dim3(b.dzblk), dim3(256), 0, s, q);
      else hipLaunchKernelGGL(linear_dz_kernel<float>, dim3(b.dzblk), dim3(256), 0, s, q);
    }
    if (dx && dw && dtype == PLYOLO_BF16 && tx == b.tile && dx_direct == dw_direct) {
      const hipError_t e = tx == 128 ? (dx_direct ? launch_both<128, true>(px, pw, gx, gw, s) : launch_both<128, false>(px, pw, gx, gw, s))
                                     : (dx_direct ? launch_both<64, true>(px, pw, gx, gw, s) : launch_both<64, false>(px, pw, gx, gw, s));
      if (e != hipSuccess) return e;
    } else {
      if (dx)
        if (hipError_t e = launch_gemm<MODE_DX>(dtype, px, tx, gx, dx_direct, s); e != hipSuccess) return e;
      if (dw)
        if (hipError_t e = launch_gemm<MODE_DW>(dtype, pw, b.tile, gw, dw_direct, s); e != hipSuccess) return e;
    }
    if (dw || db) hipLaunchKernelGGL(linear_fold_kernel, dim3((unsigned)(fw.blocks + fb.blocks)), dim3(256), 0, s, fw, fb, acc);
    return hipGetLastError();
  });
}

}  // extern "C"
