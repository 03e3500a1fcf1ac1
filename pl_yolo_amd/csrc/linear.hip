// Linear layer (1x1 convolution with bias) with activation and shortcut in its epilogue, forward and backward.
//
//   z = x . w^T + bias,  y = act(z) + res          x [M][K], w [N][K], y, z [M][N]
//   dz = dy act'(z),  dx = dz . w,  dw = dz^T . x,  db = sum over rows of dz
//
// All three products are one kernel body over two operands that are either contiguous along the contraction (KC: x and w of the forward,
// dz of dx) or along the output (RC: w of dx, dz and x of dw); an RC operand is transposed on its way out of LDS (ds_read_b64_tr_b16 in bf16).
// The product is formed as D = B . A^T, so that a lane of the MFMA result holds four consecutive COLUMNS of one output row and the epilogue
// moves 8- (bf16) or 16-byte (fp32) pieces of rows.
//
// dw contracts over the rows of the batch: the rows are split over workgroups, every range leaves a private fp32 slab and the slabs are
// added in a fixed order.
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
  int act, accumulate, vec4;
  int nj;              // column tiles
  int ksteps;          // contraction steps per slab (MODE_DW), all of them otherwise
};

// ------------------------------------------------------------------------------------------------ bf16
constexpr int BK = 64;           // contraction elements per stage
constexpr int TI = 128, TJ = 128;
typedef u32x4 __attribute__((aligned(2))) u32x4_any;     // 16 bytes at any element address
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
DEVINL s16x4 tr_read(const unsigned char* p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p); }

// eight consecutive elements of which `n` exist (the others are zero)
DEVINL u32x4 load8(const bf16_t* p, int n) {
  if (n >= 8) return *(const u32x4_any*)p;
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) v[e >> 1] |= (unsigned)p[e] << (16 * (e & 1));
  return v;
}

// One operand tile: T rows (output index) x 64 (contraction).
// KC image: [T][64] elements, 128-byte rows of eight 16-byte granules, granule g of row r at position g ^ (r & 7).
// RC image: [64][T] elements, rows of T / 16 32-byte segments, segment s of row k at position s ^ f(k): the 16 rows that one transposed read
// of a wave touches spread over all banks.
template <bool RC, int T> struct Tile {
  static constexpr int NG = T * BK / 8 / 256;      // 16-byte granules per thread
  static constexpr int BYTES = T * BK * 2;
  static DEVINL int swz(int k) { return (T >= 128 ? (k & 3) | ((k >> 1) & 4) : (k & 3)); }
  static DEVINL void request(u32x4 (&v)[NG], const bf16_t* base, int ld, int row0, int rows, int k0, int kend) {
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      const int idx = threadIdx.x + u * 256;
      if (RC) {
        const int k = k0 + idx / (T / 8), r = row0 + (idx % (T / 8)) * 8;
        const int n = k < kend ? rows - r : 0;
        v[u] = n > 0 ? load8(base + (size_t)k * ld + r, n) : u32x4{0u, 0u, 0u, 0u};
      } else {
        const int r = row0 + idx / 8, k = k0 + (idx % 8) * 8;
        const int n = r < rows ? kend - k : 0;
        v[u] = n > 0 ? load8(base + (size_t)r * ld + k, n) : u32x4{0u, 0u, 0u, 0u};
      }
    }
  }
  static DEVINL void commit(const u32x4 (&v)[NG], unsigned char* img) {
#pragma unroll
    for (int u = 0; u < NG; ++u) {
      const int idx = threadIdx.x + u * 256;
      if (RC) {
        const int k = idx / (T / 8), g = idx % (T / 8);
        *(u32x4*)(img + k * (T * 2) + (((g >> 1) ^ swz(k)) << 5) + ((g & 1) << 4)) = v[u];
      } else {
        const int r = idx / 8, g = idx % 8;
        *(u32x4*)(img + r * 128 + ((g ^ (r & 7)) << 4)) = v[u];
      }
    }
  }
  // fragment of 16 output indices starting at r0, 32 contraction elements of half kk
  static DEVINL s16x8 frag(const unsigned char* img, int r0, int kk) {
    const int lane = threadIdx.x & 63, g4 = lane >> 4, i16 = lane & 15;
    if (RC) {
      const int k = kk * 32 + 8 * g4 + (i16 >> 2), seg = r0 >> 4;
      const unsigned char* p = img + k * (T * 2) + ((seg ^ swz(k)) << 5) + ((i16 & 3) << 3);
      const s16x4 lo = tr_read(p), hi = tr_read(p + 4 * (T * 2));       // (swz(k + 4) == swz(k))
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    const int r = r0 + i16, g = kk * 4 + g4;
    return *(const s16x8*)(img + r * 128 + ((g ^ (r & 7)) << 4));
  }
};

// four consecutive columns j.. of output row i; nv of them exist
template <int MODE> DEVINL void store4(const LinP& p, int i, int j, f32x4 v) {
  const int nv = p.J - j;
  if (i >= p.I || nv <= 0) return;
  if (MODE == MODE_DW) {
    float* o = (float*)p.out + ((size_t)blockIdx.y * p.I + i) * p.J + j;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < nv) o[e] = v[e];
    return;
  }
  const bool whole = p.vec4 && nv >= 4;
  if (MODE == MODE_FWD) {
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < nv) v[e] += p.bias[j + e];
    }
    if (p.z) {
      bf16_t* z = (bf16_t*)p.z + (size_t)i * p.z_ld + j;
      if (whole) *(uint2*)z = make_uint2(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]));
      else
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < nv) z[e] = f2bf(v[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = act_fwd(v[e], p.act);
  }
  bf16_t* o = (bf16_t*)p.out + (size_t)i * p.o_ld + j;
  const bf16_t* r = MODE == MODE_FWD ? (p.res ? (const bf16_t*)p.res + (size_t)i * p.r_ld + j : nullptr) : (p.accumulate ? o : nullptr);
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

template <int MODE> __global__ __launch_bounds__(256) void linear_bf16_kernel(const LinP p) {
  constexpr bool ARC = MODE == MODE_DW, BRC = MODE != MODE_FWD;
  typedef Tile<ARC, TI> TA;
  typedef Tile<BRC, TJ> TB;
  __shared__ __align__(16) unsigned char smem[2][TA::BYTES + TB::BYTES];
  const int i0 = (int)(blockIdx.x / p.nj) * TI, j0 = (int)(blockIdx.x % p.nj) * TJ;
  const int wave = threadIdx.x >> 6, wi = (wave >> 1) * 64, wj = (wave & 1) * 64;
  const int kbeg = MODE == MODE_DW ? (int)blockIdx.y * p.ksteps * BK : 0;
  const int kend = MODE == MODE_DW ? min(p.Kc, kbeg + p.ksteps * BK) : p.Kc;
  f32x4 acc[4][4];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  u32x4 va[TA::NG], vb[TB::NG];
  TA::request(va, (const bf16_t*)p.a, p.a_ld, i0, p.I, kbeg, kend);
  TB::request(vb, (const bf16_t*)p.b, p.b_ld, j0, p.J, kbeg, kend);
  int buf = 0;
  for (int k0 = kbeg; k0 < kend; k0 += BK, buf ^= 1) {
    unsigned char *ia = smem[buf], *ib = smem[buf] + TA::BYTES;
    TA::commit(va, ia);
    TB::commit(vb, ib);
    __syncthreads();      // image `buf` is whole; image buf ^ 1 was last read before every wave came here
    if (k0 + BK < kend) {
      TA::request(va, (const bf16_t*)p.a, p.a_ld, i0, p.I, k0 + BK, kend);
      TB::request(vb, (const bf16_t*)p.b, p.b_ld, j0, p.J, k0 + BK, kend);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      s16x8 fa[4], fb[4];
#pragma unroll
      for (int a = 0; a < 4; ++a) fa[a] = TA::frag(ia, wi + a * 16, kk);
#pragma unroll
      for (int b = 0; b < 4; ++b) fb[b] = TB::frag(ib, wj + b * 16, kk);
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b)
          acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8*)&fb[b], *(const bf16x8*)&fa[a], acc[a][b], 0, 0, 0);
    }
  }
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) store4<MODE>(p, i0 + wi + a * 16 + (lane & 15), j0 + wj + b * 16 + 4 * (lane >> 4), acc[a][b]);
}

// ------------------------------------------------------------------------------------------------ fp32 (parity mode)
// 64 x 64 tile, four waves of 32 x 32 (2 x 2 fragments of v_mfma_f32_16x16x4_f32), 16 contraction elements per stage; both LDS images are
// [k][row] with a pitch of 80 floats: the four k rows of one fragment read start 16 banks apart.
constexpr int FT = 64, FK = 16, FP = 80;

template <bool RC> DEVINL void f32_request(float (&v)[4], const float* base, int ld, int row0, int rows, int k0, int kend) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int idx = threadIdx.x + u * 256;
    const int k = k0 + (RC ? idx / FT : idx % FK), r = row0 + (RC ? idx % FT : idx / FK);
    v[u] = (k < kend && r < rows) ? base[RC ? (size_t)k * ld + r : (size_t)r * ld + k] : 0.f;
  }
}
template <bool RC> DEVINL void f32_commit(const float (&v)[4], float* img) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int idx = threadIdx.x + u * 256;
    img[(RC ? idx / FT : idx % FK) * FP + (RC ? idx % FT : idx / FK)] = v[u];
  }
}

template <int MODE> __global__ __launch_bounds__(256) void linear_f32_kernel(const LinP p) {
  constexpr bool ARC = MODE == MODE_DW, BRC = MODE != MODE_FWD;
  __shared__ float smem[2][2 * FK * FP];
  const int i0 = (int)(blockIdx.x / p.nj) * FT, j0 = (int)(blockIdx.x % p.nj) * FT;
  const int wave = threadIdx.x >> 6, wi = (wave >> 1) * 32, wj = (wave & 1) * 32, lane = threadIdx.x & 63;
  const int kbeg = MODE == MODE_DW ? (int)blockIdx.y * p.ksteps * FK : 0;
  const int kend = MODE == MODE_DW ? min(p.Kc, kbeg + p.ksteps * FK) : p.Kc;
  f32x4 acc[2][2];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  float va[4], vb[4];
  f32_request<ARC>(va, (const float*)p.a, p.a_ld, i0, p.I, kbeg, kend);
  f32_request<BRC>(vb, (const float*)p.b, p.b_ld, j0, p.J, kbeg, kend);
  int buf = 0;
  for (int k0 = kbeg; k0 < kend; k0 += FK, buf ^= 1) {
    float *ia = smem[buf], *ib = smem[buf] + FK * FP;
    f32_commit<ARC>(va, ia);
    f32_commit<BRC>(vb, ib);
    __syncthreads();
    if (k0 + FK < kend) {
      f32_request<ARC>(va, (const float*)p.a, p.a_ld, i0, p.I, k0 + FK, kend);
      f32_request<BRC>(vb, (const float*)p.b, p.b_ld, j0, p.J, k0 + FK, kend);
    }
#pragma unroll
    for (int kk = 0; kk < FK / 4; ++kk) {
      const int ro = (kk * 4 + (lane >> 4)) * FP + (lane & 15);
      float fa[2], fb[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) fa[a] = ia[ro + wi + a * 16];
#pragma unroll
      for (int b = 0; b < 2; ++b) fb[b] = ib[ro + wj + b * 16];
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[b], fa[a], acc[a][b], 0, 0, 0);
    }
  }
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int i = i0 + wi + a * 16 + (lane & 15), j = j0 + wj + b * 16 + 4 * (lane >> 4);
      if (i >= p.I) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (j + e >= p.J) continue;
        float v = acc[a][b][e];
        if (MODE == MODE_DW) {
          ((float*)p.out)[((size_t)blockIdx.y * p.I + i) * p.J + j + e] = v;
          continue;
        }
        float* o = (float*)p.out + (size_t)i * p.o_ld + j + e;
        if (MODE == MODE_FWD) {
          if (p.bias) v += p.bias[j + e];
          if (p.z) ((float*)p.z)[(size_t)i * p.z_ld + j + e] = v;
          v = act_fwd_precise(v, p.act);
          if (p.res) v += ((const float*)p.res)[(size_t)i * p.r_ld + j + e];
        } else if (p.accumulate) {
          v += *o;
        }
        *o = v;
      }
    }
}

// ------------------------------------------------------------------------------------------------ dz, db, slab sums
struct DzP {
  const void* dy;
  const void* z;        // NULL: dz = dy (only the column sums are formed)
  void* dz;             // [M][dz_ld], columns N .. dz_ld zero; NULL with z
  float* part;          // [blocks][N] column sums, or NULL
  int M, N, dy_ld, z_ld, dz_ld, act, rows;
};

// 64 columns x 4 row lanes per workgroup, `rows` rows
template <typename T> __global__ __launch_bounds__(256) void linear_dz_kernel(const DzP p) {
  const int c = (int)blockIdx.x * 64 + (threadIdx.x & 63), rl = threadIdx.x >> 6;
  const int64_t m0 = (int64_t)blockIdx.y * p.rows;
  const int64_t m1 = min((int64_t)p.M, m0 + p.rows);
  float s = 0.f;
  for (int64_t m = m0 + rl; m < m1; m += 4) {
    float d = 0.f;
    if (c < p.N) {
      d = ActT<T>::ld((const T*)p.dy + (size_t)m * p.dy_ld + c);
      if (p.z) d *= act_grad<Vec<T>::precise>(ActT<T>::ld((const T*)p.z + (size_t)m * p.z_ld + c), p.act);
      s += d;
    }
    if (p.dz && c < p.dz_ld) ActT<T>::st((T*)p.dz + (size_t)m * p.dz_ld + c, d);
  }
  __shared__ float red[256];
  red[threadIdx.x] = s;
  __syncthreads();
  if (rl == 0 && c < p.N && p.part) p.part[(size_t)blockIdx.y * p.N + c] = (s + red[threadIdx.x + 64]) + (red[threadIdx.x + 128] + red[threadIdx.x + 192]);
}

// out[e] (+)= sum over S slabs of part[s][e], in order; 64 elements x 4 slab lanes per workgroup
template <typename O> __global__ __launch_bounds__(256) void linear_fold_kernel(const float* part, int S, size_t elems, O* out, int accumulate) {
  const size_t e = (size_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const int sl = threadIdx.x >> 6;
  float v = 0.f;
  if (e < elems)
    for (int s = sl; s < S; s += 4) v += part[(size_t)s * elems + e];
  __shared__ float red[256];
  red[threadIdx.x] = v;
  __syncthreads();
  if (sl == 0 && e < elems) {
    v = (v + red[threadIdx.x + 64]) + (red[threadIdx.x + 128] + red[threadIdx.x + 192]);
    if (accumulate) v += ActT<O>::ld(out + e);
    ActT<O>::st(out + e, v);
  }
}

// ------------------------------------------------------------------------------------------------ host side
constexpr int DZ_ROWS = 256;     // rows per workgroup of linear_dz_kernel (more where that would make over 4096 of them)

struct BwdPlan {
  int dz_ld, S, ksteps, dzblk, dzrows;
  size_t dz_bytes, part_off, part_bytes, slab_off, slab_bytes, total;
};

size_t up16(size_t v) { return (v + 15) & ~(size_t)15; }

// Slabs of dw: enough row ranges to give every compute unit a workgroup, at least four stages each.
BwdPlan bwd_plan(const plyolo_linear_desc* d) {
  BwdPlan b{};
  const bool half = d->dtype == PLYOLO_BF16;
  const int es = half ? 2 : 4, ti = half ? TI : FT, bk = half ? BK : FK;
  b.dz_ld = (d->N + 7) & ~7;
  b.dz_bytes = d->act == PLYOLO_ACT_NONE ? 0 : up16((size_t)d->M * b.dz_ld * es);
  b.dzrows = max(DZ_ROWS, cdiv(d->M, 4096));
  b.dzblk = cdiv(d->M, b.dzrows);
  b.part_off = b.dz_bytes;
  b.part_bytes = up16((size_t)b.dzblk * d->N * 4);
  b.slab_off = b.part_off + b.part_bytes;
  const int64_t tiles = (int64_t)cdiv(d->N, ti) * cdiv(d->K, ti);
  const int steps = cdiv(d->M, bk);
  int64_t s = (256 + tiles - 1) / tiles;
  if (s > (steps + 3) / 4) s = (steps + 3) / 4;
  if (s < 1) s = 1;
  b.ksteps = (int)((steps + s - 1) / s);
  b.S = (steps + b.ksteps - 1) / b.ksteps;
  b.slab_bytes = up16((size_t)b.S * d->N * d->K * 4);
  b.total = b.slab_off + b.slab_bytes;
  return b;
}

int check_linear(const plyolo_linear_desc* d, const char* who) {
  PLY_CHECK_ARG(d != nullptr, "%s: null descriptor", who);
  PLY_CHECK_ARG(d->dtype == PLYOLO_BF16 || d->dtype == PLYOLO_F32, "%s: bad dtype %d", who, d->dtype);
  PLY_CHECK_ARG(d->M > 0 && d->N > 0 && d->K > 0, "%s: non-positive dimension (M %d, N %d, K %d)", who, d->M, d->N, d->K);
  PLY_CHECK_ARG(d->N <= (1 << 20) && d->K <= (1 << 20) && d->M <= 2147483647 - 1024, "%s: dimension too large (M %d, N %d, K %d)", who, d->M, d->N, d->K);
  PLY_CHECK_ARG(d->act >= PLYOLO_ACT_NONE && d->act <= PLYOLO_ACT_GELU, "%s: bad activation %d", who, d->act);
  PLY_CHECK_ARG(d->x_ld >= d->K && d->w_ld >= d->K, "%s: x_ld %d or w_ld %d < K %d", who, d->x_ld, d->w_ld, d->K);
  return 0;
}

// tile grid of an I x J output; the column tiles of one row tile are neighbours, so that its rows are read from HBM once
int tile_grid(LinP& p, int t, const char* who) {
  p.nj = cdiv(p.J, t);
  const int64_t n = (int64_t)cdiv(p.I, t) * p.nj;
  PLY_CHECK_ARG(n < 2147483647, "%s: more than 2^31 tiles", who);
  return (int)n;
}

template <int MODE> hipError_t launch_gemm(int dtype, const LinP& p, int grid, int slabs, hipStream_t s) {
  if (dtype == PLYOLO_BF16) hipLaunchKernelGGL(linear_bf16_kernel<MODE>, dim3(grid, slabs), dim3(256), 0, s, p);
  else hipLaunchKernelGGL(linear_f32_kernel<MODE>, dim3(grid, slabs), dim3(256), 0, s, p);
  return hipGetLastError();
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
  const int grid = tile_grid(p, dtype == PLYOLO_BF16 ? TI : FT, "linear_fwd");
  if (grid < 0) return -1;
  const double m = d->M, n = d->N, k = d->K;
  plyolo::annotate("linear_fwd", 2.0 * m * n * k, (m * k + n * k + m * n * (1.0 + (z ? 1 : 0) + (res ? 1 : 0))) * es);
  return plyolo::submit(stream, [=](hipStream_t s) -> hipError_t { return launch_gemm<MODE_FWD>(dtype, p, grid, 1, s); });
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
  px.a = g; px.b = w; px.out = dx; px.I = d->M; px.J = d->K; px.Kc = d->N;
  px.a_ld = g_ld; px.b_ld = d->w_ld; px.o_ld = dx_ld; px.accumulate = accumulate_dx ? 1 : 0;
  px.vec4 = dx_ld % 4 == 0 && (size_t)dx % 8 == 0;
  pw.a = g; pw.b = x; pw.out = ws + b.slab_off; pw.I = d->N; pw.J = d->K; pw.Kc = d->M;
  pw.a_ld = g_ld; pw.b_ld = d->x_ld; pw.ksteps = b.ksteps;
  const int t = dtype == PLYOLO_BF16 ? TI : FT;
  const int gx = tile_grid(px, t, "linear_bwd"), gw = tile_grid(pw, t, "linear_bwd");
  if (gx < 0 || gw < 0) return -1;
  const size_t elems = (size_t)d->N * d->K;
  const int N = d->N, acc = accumulate_params ? 1 : 0;
  const dim3 dzgrid(cdiv(has_act ? b.dz_ld : d->N, 64), b.dzblk);
  const double m = d->M, n = d->N, k = d->K;
  plyolo::annotate("linear_bwd", 2.0 * m * n * k * ((dx ? 1 : 0) + (dw ? 1 : 0)), (m * n * (has_act ? 2.0 : 1.0) + 2.0 * m * k + 2.0 * n * k) * es);
  return plyolo::submit(stream, [=](hipStream_t s) -> hipError_t {
    if (q.dz || q.part) {
      if (dtype == PLYOLO_BF16) hipLaunchKernelGGL(linear_dz_kernel<bf16_t>, dzgrid, dim3(256), 0, s, q);
      else hipLaunchKernelGGL(linear_dz_kernel<float>, dzgrid, dim3(256), 0, s, q);
    }
    if (db) hipLaunchKernelGGL(linear_fold_kernel<float>, dim3((unsigned)cdiv(N, 64)), dim3(256), 0, s, q.part, b.dzblk, (size_t)N, db, acc);
    if (dx)
      if (hipError_t e = launch_gemm<MODE_DX>(dtype, px, gx, 1, s); e != hipSuccess) return e;
    if (dw) {
      if (hipError_t e = launch_gemm<MODE_DW>(dtype, pw, gw, b.S, s); e != hipSuccess) return e;
      const dim3 fg((unsigned)cdivz(elems, 64));
      if (dw_dtype == PLYOLO_F32) hipLaunchKernelGGL(linear_fold_kernel<float>, fg, dim3(256), 0, s, (const float*)pw.out, b.S, elems, (float*)dw, acc);
      else hipLaunchKernelGGL(linear_fold_kernel<bf16_t>, fg, dim3(256), 0, s, (const float*)pw.out, b.S, elems, (bf16_t*)dw, acc);
    }
    return hipGetLastError();
  });
}

}  // extern "C"
