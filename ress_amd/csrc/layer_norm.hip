// Layer norm over the last dim, its backward pass, and both of a residual sum h = x + gamma * branch.
//
//   n = (h - mean) rstd w + b,  rstd = 1 / sqrt(var + eps);   with g = dn w, xh = (h - mean) rstd:
//   dh += rstd (g - mean(g) - xh mean(g xh)),  dw = sum over rows of dn xh,  db = of dn,  dbranch = gamma dh,  dgamma = of dh branch
//
// A row's elements stay in the registers of TPR threads, K pieces of 8 each; mean and variance are taken one after the other
// from there, in fp32. The weights' gradients are summed row by row in registers, over a workgroup's threads of the same column in
// LDS, and over the workgroups by a second kernel, all in a fixed order. Bound by the bytes: a workgroup goes through
// many rows, so that the weights are read and the sums are written a few hundred times and not once a row, and a row's loads are in
// flight while the row before is computed. 21,984 rows of 1,024 in bf16, residual sum and LayerScale included: forward 33 us
// (180 MB, 5.5 TB/s; without the loads ahead 45), backward 47 (270 MB, 5.8 TB/s; 80) and 4 for the parts' sums. Four waves a
// workgroup and 512 workgroups; eight waves 35 + 48, half the workgroups 34 + 47, twice as many 35 + 49. Rows that cannot be read
// 16 bytes at a time go element by element, without a branch between the loads: 9,470 rows of 1,637 in fp32, residual sum
// included, forward 44 us and backward 54 (with one 138 and 259), in bf16 30 and 48.
#include "../../include/ress_hip.h"
#include "common.h"

namespace {

enum { LN_F32 = 0, LN_BF16 = 1, LN_F16 = 2 };
constexpr int LN_MOST = 8192;
constexpr int LN_GROUPS = 512;  // workgroups at most: the weights' gradients have that many parts

struct Rows {  // rows (i0, i1, i2) of unit-stride elements
  char* p;
  long long s0, s1, s2;  // bytes
};
struct NormArgs {
  Rows x, branch, dn, dh;
  char *sum, *out, *dx, *dbranch;  // contiguous rows
  const void *gamma, *weight, *bias;
  int n1, n2, C;
  long long rows;
  float eps;
  int wide;              // weights in fp32
  float *mean, *rstd;
  float* part;           // [workgroup][3][C]: dw, db, dgamma
};

__device__ __forceinline__ const char* row_of(const Rows& r, long long i, const NormArgs& a) {
  if (a.n1 == 1 && a.n2 == 1) return r.p + i * r.s0;
  const unsigned q = (unsigned)(i / a.n2), i2 = (unsigned)(i - (long long)q * a.n2);
  return r.p + (long long)(q / (unsigned)a.n1) * r.s0 + (long long)(q % (unsigned)a.n1) * r.s1 + (long long)i2 * r.s2;
}
template <int DT>
constexpr int bytes_of() { return DT == LN_F32 ? 4 : 2; }
template <int DT>
__device__ __forceinline__ float to_f32(uint32_t bits) {
  if constexpr (DT == LN_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  else return __uint_as_float(bits << 16);
}
template <int DT>
__device__ __forceinline__ uint32_t bits16(float x) {
  if constexpr (DT == LN_F16) return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x);
  else return f32_to_bf16_bits(x);
}
template <int DT>
__device__ __forceinline__ float rounded(float x) {
  if constexpr (DT == LN_F32) return x;
  else return to_f32<DT>(bits16<DT>(x));
}

// Where thread t of a row's TPR has piece k's element u: eight neighbours (VEC: C a multiple of 8, rows 16-byte aligned), or
// neighbours in neighbouring threads.
template <int TPR, bool VEC>
__device__ __forceinline__ int place(int t, int k, int u) {
  return VEC ? (k * TPR + t) * 8 + u : (k * 8 + u) * TPR + t;
}
// Piece k of a row as it is loaded, and its values (zeros past the row's end)
template <int DT, int TPR, bool VEC>
struct Piece {
  // 16-bit elements that come by themselves stay in a register each (packing would wait for them) where there are enough
  static constexpr int N = DT == LN_F32 || (!VEC && TPR < 1024) ? 2 : 1;
  uint4 v[N];
  __device__ __forceinline__ void load(const char* row, int t, int k, int C) {
    if constexpr (VEC) {
      const int at = place<TPR, true>(t, k, 0);
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = at < C ? reinterpret_cast<const uint4*>(row)[at / 8 * N + i] : make_uint4(0, 0, 0, 0);
    } else {
      uint32_t x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int at = min(place<TPR, false>(t, k, u), C - 1);  // no branch between the loads
        x[u] = DT == LN_F32 ? reinterpret_cast<const uint32_t*>(row)[at] : reinterpret_cast<const uint16_t*>(row)[at];
      }
      if constexpr (N == 2) {
        v[0] = make_uint4(x[0], x[1], x[2], x[3]);
        v[1] = make_uint4(x[4], x[5], x[6], x[7]);
      } else {
        v[0] = make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
      }
    }
  }
  __device__ __forceinline__ void values(int t, int k, int C, float (&x)[8]) const {
    if constexpr (N == 2) {
      const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[N - 1].x, v[N - 1].y, v[N - 1].z, v[N - 1].w};
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = DT == LN_F32 ? __uint_as_float(w[u]) : to_f32<DT>(w[u]);
    } else {
      const uint32_t w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = to_f32<DT>(u & 1 ? w[u >> 1] >> 16 : w[u >> 1] & 0xffffu);
    }
    if constexpr (!VEC) {
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = place<TPR, false>(t, k, u) < C ? x[u] : 0.0f;
    }
  }
};
template <int DT, int TPR, bool VEC>
__device__ __forceinline__ void load8(const char* row, int t, int k, int C, float (&x)[8]) {
  Piece<DT, TPR, VEC> p;
  p.load(row, t, k, C);
  p.values(t, k, C, x);
}
template <int DT, int TPR, bool VEC>
__device__ __forceinline__ void store8(char* row, int t, int k, int C, const float (&x)[8]) {
  if constexpr (VEC) {
    const int at = place<TPR, true>(t, k, 0);
    if (at >= C) return;
    if constexpr (DT == LN_F32) {
      reinterpret_cast<float4*>(row)[at / 4] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(row)[at / 4 + 1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      uint32_t v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = bits16<DT>(x[2 * i]) | bits16<DT>(x[2 * i + 1]) << 16;
      reinterpret_cast<uint4*>(row)[at / 8] = make_uint4(v[0], v[1], v[2], v[3]);
    }
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int at = place<TPR, false>(t, k, u);
      if (at >= C) continue;
      if constexpr (DT == LN_F32) reinterpret_cast<float*>(row)[at] = x[u];
      else reinterpret_cast<uint16_t*>(row)[at] = (uint16_t)bits16<DT>(x[u]);
    }
  }
}
// a weight's piece, `none` where there is no weight; the pointers are as aligned as the rows (VEC)
template <int DT, int TPR, bool VEC>
__device__ __forceinline__ void load_weight(const void* w, int wide, float none, int t, int k, int C, float (&x)[8]) {
  if (!w) {
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = none;
  } else if (wide) {
    load8<LN_F32, TPR, VEC>(reinterpret_cast<const char*>(w), t, k, C, x);
  } else {
    load8<DT, TPR, VEC>(reinterpret_cast<const char*>(w), t, k, C, x);
  }
}

// Sums over a row's threads, in every one of them
template <int TPR>
__device__ __forceinline__ void row_sums(float& a, float& b, float* lds) {
  constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
  for (int s = 1; s < W; s <<= 1) {
    a += __shfl_xor(a, s, 64);
    b += __shfl_xor(b, s, 64);
  }
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    __syncthreads();  // the row before is done with lds
    if ((threadIdx.x & 63) == 0) {
      lds[threadIdx.x >> 6] = a;
      lds[NW + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      a += lds[i];
      b += lds[NW + i];
    }
  }
}
constexpr int ln_threads(int TPR) { return TPR > 256 ? TPR : 256; }
// A thread's row of its workgroup's; where a wave has one row alone the compiler shall know it, and keep addresses in scalar registers
template <int TPR>
__device__ __forceinline__ int row_in_group() {
  if constexpr (TPR >= 256) return 0;
  else if constexpr (TPR >= 64) return __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
  else return threadIdx.x / TPR;
}

template <int DT, int TPR, int K, bool VEC>
__global__ __launch_bounds__(ln_threads(TPR)) void k_layer_norm_fwd(NormArgs a) {
  constexpr int NT = ln_threads(TPR), RPG = NT / TPR, SZ = bytes_of<DT>();
  __shared__ float lds[TPR > 64 ? 2 * (TPR / 64) : 1];
  const int t = threadIdx.x % TPR;
  float w[K][8], b[K][8], gm[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    load_weight<DT, TPR, VEC>(a.weight, a.wide, 1.0f, t, k, a.C, w[k]);
    load_weight<DT, TPR, VEC>(a.bias, a.wide, 0.0f, t, k, a.C, b[k]);
    load_weight<DT, TPR, VEC>(a.gamma, a.wide, 1.0f, t, k, a.C, gm[k]);
  }
  const float inv = 1.0f / (float)a.C;
  // a row's loads go out while the one before is computed
  Piece<DT, TPR, VEC> px[K], pb[K];
  auto load = [&](long long r) {
    const char* xr = row_of(a.x, r, a);
#pragma unroll
    for (int k = 0; k < K; ++k) px[k].load(xr, t, k, a.C);
    if (a.branch.p) {
      const char* br = row_of(a.branch, r, a);
#pragma unroll
      for (int k = 0; k < K; ++k) pb[k].load(br, t, k, a.C);
    }
  };
  const long long step = (long long)gridDim.x * RPG;
  long long r = (long long)blockIdx.x * RPG + row_in_group<TPR>();
  if (r < a.rows) load(r);
  for (; r < a.rows; r += step) {  // a row's threads go together, and only they wait for each other
    float x[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k) px[k].values(t, k, a.C, x[k]);
    if (a.branch.p) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float y[8];
        pb[k].values(t, k, a.C, y);
        // the norm is that of the sum as it is returned, and the backward pass reads that
#pragma unroll
        for (int u = 0; u < 8; ++u) x[k][u] = rounded<DT>(fmaf(gm[k][u], y[u], x[k][u]));
        store8<DT, TPR, VEC>(a.sum + r * a.C * SZ, t, k, a.C, x[k]);
      }
    }
    if (r + step < a.rows) load(r + step);
    float s = 0.0f, none = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int u = 0; u < 8; ++u) s += x[k][u];
    row_sums<TPR>(s, none, lds);
    const float mean = s * inv;
    float v = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        x[k][u] = place<TPR, VEC>(t, k, u) < a.C ? x[k][u] - mean : 0.0f;
        v = fmaf(x[k][u], x[k][u], v);
      }
    row_sums<TPR>(v, none, lds);
    const float rstd = 1.0f / sqrtf(v * inv + a.eps);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int u = 0; u < 8; ++u) x[k][u] = fmaf(x[k][u] * rstd, w[k][u], b[k][u]);
      store8<DT, TPR, VEC>(a.out + r * a.C * SZ, t, k, a.C, x[k]);
    }
    if (a.mean && t == 0) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
  }
}

// x: the rows that were normalised (the sum, if there is a branch)
template <int DT, int TPR, int K, bool VEC>
__global__ __launch_bounds__(ln_threads(TPR)) void k_layer_norm_bwd(NormArgs a) {
  constexpr int NT = ln_threads(TPR), RPG = NT / TPR, SZ = bytes_of<DT>(), COLS = TPR * K * 8;
  constexpr bool AHEAD = TPR < 1024;  // 128 registers a lane are too few for a row's loads beside the row before (692 us for 896)
  constexpr int PER = TPR <= 64 ? NT / 64 : 1;  // parts of a column in the workgroup: one a wave
  __shared__ float lds[TPR > 64 ? 2 * (TPR / 64) : PER * COLS];
  const int t = threadIdx.x % TPR;
  float w[K][8], gm[K][8], dw[K][8], db[K][8], dg[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    load_weight<DT, TPR, VEC>(a.weight, a.wide, 1.0f, t, k, a.C, w[k]);
    load_weight<DT, TPR, VEC>(a.gamma, a.wide, 1.0f, t, k, a.C, gm[k]);
#pragma unroll
    for (int u = 0; u < 8; ++u) dw[k][u] = db[k][u] = dg[k][u] = 0.0f;
  }
  const float inv = 1.0f / (float)a.C;
  Piece<DT, TPR, VEC> px[K], pn[K], ph[K], pb[K];
  float mean = 0.0f, rstd = 0.0f;
  auto load = [&](long long r) {
    mean = a.mean[r];
    rstd = a.rstd[r];
    auto row = [&](Piece<DT, TPR, VEC> (&p)[K], const Rows& rows) {
      if (!rows.p) return;
      const char* at = row_of(rows, r, a);
#pragma unroll
      for (int k = 0; k < K; ++k) p[k].load(at, t, k, a.C);
    };
    row(px, a.x);
    row(pn, a.dn);
    row(ph, a.dh);
    row(pb, a.branch);
  };
  const long long step = (long long)gridDim.x * RPG;
  long long r = (long long)blockIdx.x * RPG + row_in_group<TPR>();
  if (AHEAD && r < a.rows) load(r);
  for (; r < a.rows; r += step) {
    if (!AHEAD) load(r);
    float xh[K][8], g[K][8], more[K][8], y[K][8];
    const float m = mean, rs = rstd;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      px[k].values(t, k, a.C, xh[k]);
      if (a.dn.p) pn[k].values(t, k, a.C, g[k]);
      if (a.dh.p) ph[k].values(t, k, a.C, more[k]);
      if (a.branch.p) pb[k].values(t, k, a.C, y[k]);
    }
    if (AHEAD && r + step < a.rows) load(r + step);
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int u = 0; u < 8; ++u) {  // past the row's end g is 0
        if (!a.dn.p) g[k][u] = 0.0f;
        xh[k][u] = (xh[k][u] - m) * rs;
        dw[k][u] = fmaf(g[k][u], xh[k][u], dw[k][u]);
        db[k][u] += g[k][u];
        g[k][u] *= w[k][u];
        s1 += g[k][u];
        s2 = fmaf(g[k][u], xh[k][u], s2);
      }
    row_sums<TPR>(s1, s2, lds);
    s1 *= inv;
    s2 *= inv;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        g[k][u] = rs * (g[k][u] - fmaf(xh[k][u], s2, s1));
        if (a.dh.p) g[k][u] += more[k][u];
      }
      if (a.dx) store8<DT, TPR, VEC>(a.dx + r * a.C * SZ, t, k, a.C, g[k]);
      if (a.branch.p) {
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          dg[k][u] = fmaf(g[k][u], y[k][u], dg[k][u]);
          g[k][u] *= gm[k][u];
        }
        if (a.dbranch) store8<DT, TPR, VEC>(a.dbranch + r * a.C * SZ, t, k, a.C, g[k]);
      }
    }
  }
  if (!a.part) return;
  float* to = a.part + (long long)blockIdx.x * 3 * a.C;
#pragma unroll
  for (int which = 0; which < 3; ++which) {
    if (which == 2 && !a.branch.p) break;
    float (&acc)[K][8] = which == 0 ? dw : which == 1 ? db : dg;
    if constexpr (TPR > 64) {
#pragma unroll
      for (int k = 0; k < K; ++k) store8<LN_F32, TPR, VEC>(reinterpret_cast<char*>(to + which * a.C), t, k, a.C, acc[k]);
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int u = 0; u < 8; ++u) {
#pragma unroll
          for (int s = TPR; s < 64; s <<= 1) acc[k][u] += __shfl_xor(acc[k][u], s, 64);
          if ((threadIdx.x & 63) < TPR) lds[(threadIdx.x >> 6) * COLS + place<TPR, VEC>(t, k, u)] = acc[k][u];
        }
      __syncthreads();
      for (int c = threadIdx.x; c < a.C; c += NT) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) s += lds[i * COLS + c];
        to[which * a.C + c] = s;
      }
      __syncthreads();
    }
  }
}

// The weights' gradients: sums over the parts of 64 columns, 16 threads a column
struct Ends {
  void* to[3];
  int wide;
};
template <int DT>
__global__ __launch_bounds__(1024) void k_layer_norm_ends(const float* __restrict__ part, int parts, int C, Ends e) {
  __shared__ float lds[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), which = blockIdx.y, y = threadIdx.x >> 6;
  if (!e.to[which]) return;
  float s = 0.0f;
  if (c < C)
#pragma unroll 8
    for (int i = y; i < parts; i += 16) s += part[((long long)i * 3 + which) * C + c];
  lds[y][threadIdx.x & 63] = s;
  __syncthreads();
  if (y == 0 && c < C) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += lds[i][threadIdx.x];
    if (DT == LN_F32 || e.wide) reinterpret_cast<float*>(e.to[which])[c] = s;
    else reinterpret_cast<uint16_t*>(e.to[which])[c] = (uint16_t)bits16<DT>(s);
  }
}

// The shape that takes rows of C elements: as few threads a row as leave a thread 16 elements at most, 8 where they are loaded one by
// one (16: 1,637 in fp32 184 and 531 us). 9,470 rows of 8,000 in 512 threads for 1,024: bf16 109 + 191 us for 141 + 190, fp32 222 +
// 328 for 225 + 505.
template <class F>
void with_shape(int C, bool vec, F f) {
#define RESS_LN_SHAPE(T, K, V) f(std::integral_constant<int, T>{}, std::integral_constant<int, K>{}, std::integral_constant<bool, V>{})
  if (vec) {
    if (C <= 64) RESS_LN_SHAPE(8, 1, true);
    else if (C <= 128) RESS_LN_SHAPE(16, 1, true);
    else if (C <= 512) RESS_LN_SHAPE(64, 1, true);
    else if (C <= 1024) RESS_LN_SHAPE(64, 2, true);
    else if (C <= 2048) RESS_LN_SHAPE(256, 1, true);
    else if (C <= 4096) RESS_LN_SHAPE(256, 2, true);
    else RESS_LN_SHAPE(512, 2, true);
  } else {
    if (C <= 512) RESS_LN_SHAPE(64, 1, false);
    else if (C <= 2048) RESS_LN_SHAPE(256, 1, false);
    else if (C <= 4096) RESS_LN_SHAPE(512, 1, false);
    else RESS_LN_SHAPE(1024, 1, false);
  }
}
template <class F>
void with_type(int dtype, F f) {
  if (dtype == LN_F32) f(std::integral_constant<int, LN_F32>{});
  else if (dtype == LN_BF16) f(std::integral_constant<int, LN_BF16>{});
  else f(std::integral_constant<int, LN_F16>{});
}
int groups(long long rows, int rpg) {
  const long long n = (rows + rpg - 1) / rpg;
  return (int)(n < LN_GROUPS ? n : LN_GROUPS);
}

NormArgs arguments(const ress_layer_norm* c) {
  NormArgs a{};
  const int size = c->dtype == LN_F32 ? 4 : 2;
  auto rows = [&](const ress_rows& r) { return Rows{(char*)r.data, r.s0 * size, r.s1 * size, r.s2 * size}; };
  a.x = rows(c->x);
  a.branch = rows(c->branch);
  a.sum = (char*)c->sum;
  a.out = (char*)c->out;
  a.gamma = c->gamma;
  a.weight = c->weight;
  a.bias = c->bias;
  a.n1 = c->n1;
  a.n2 = c->n2;
  a.C = c->C;
  a.rows = (long long)c->n0 * c->n1 * c->n2;
  a.eps = c->eps;
  a.wide = c->wide || c->dtype == LN_F32;
  a.mean = c->mean;
  a.rstd = c->rstd;
  return a;
}
int check(const ress_layer_norm* c, const char* name) {
  RESS_REQUIRE(c, "%s: null arguments", name);
  RESS_REQUIRE(c->dtype >= LN_F32 && c->dtype <= LN_F16, "%s: dtype code %d", name, c->dtype);
  RESS_REQUIRE(c->n0 >= 0 && c->n1 >= 1 && c->n2 >= 1 && (long long)c->n1 * c->n2 < 1ll << 31 &&
                   (long long)c->n0 * c->n1 * c->n2 < 1ll << 31,
               "%s: bad geometry (at most 2^31 - 1 rows)", name);
  RESS_REQUIRE(c->C >= 1 && c->C <= LN_MOST, "%s: rows of %d elements (1 to %d)", name, c->C, LN_MOST);
  RESS_REQUIRE(c->eps >= 0.0f, "%s: eps must not be negative", name);
  return 0;
}
bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool aligned(const Rows& r) { return aligned(r.p) && ((r.s0 | r.s1 | r.s2) & 15) == 0; }

}  // namespace

RESS_API int ress_layer_norm_fwd(const ress_layer_norm* c, hipStream_t stream) {
  const char* name = "ress_layer_norm_fwd";
  if (int rc = check(c, name)) return rc;
  const NormArgs a = arguments(c);
  if (!a.rows) return 0;
  RESS_REQUIRE(a.x.p && a.out && (!a.branch.p || a.sum) && (!a.mean == !a.rstd), "%s: null buffer", name);
  const bool vec = a.C % 8 == 0 && aligned(a.x) && aligned(a.branch) && aligned(a.sum) && aligned(a.out) && aligned(a.gamma) &&
                   aligned(a.weight) && aligned(a.bias);
  with_type(c->dtype, [&](auto dt) {
    with_shape(a.C, vec, [&](auto tpr, auto k, auto v) {
      constexpr int T = decltype(tpr)::value, NT = ln_threads(T);
      // without sums to hand on a row more a workgroup saves nothing: four times as many
      const long long n = (a.rows + NT / T - 1) / (NT / T);
      hipLaunchKernelGGL((k_layer_norm_fwd<decltype(dt)::value, T, decltype(k)::value, decltype(v)::value>),
                         dim3((unsigned)(n < 4 * LN_GROUPS ? n : 4 * LN_GROUPS)), dim3(NT), 0, stream, a);
    });
  });
  RESS_LAUNCHED("k_layer_norm_fwd");
  return 0;
}

RESS_API long long ress_layer_norm_bwd_workspace_size(const ress_layer_norm* c) {
  if (!c || c->C < 1 || c->C > LN_MOST || c->n0 < 0 || c->n1 < 1 || c->n2 < 1) return -1;
  const long long rows = (long long)c->n0 * c->n1 * c->n2;
  return 4ll * 3 * c->C * (rows < LN_GROUPS ? rows : LN_GROUPS);  // a workgroup has at least a row
}

RESS_API int ress_layer_norm_bwd(const ress_layer_norm* c, const ress_rows* grad_out, const ress_rows* grad_sum, void* dx,
                                 void* dbranch, void* dgamma, void* dweight, void* dbias, void* workspace,
                                 long long workspace_bytes, hipStream_t stream) {
  const char* name = "ress_layer_norm_bwd";
  if (int rc = check(c, name)) return rc;
  NormArgs a = arguments(c);
  const int size = c->dtype == LN_F32 ? 4 : 2;
  if (grad_out) a.dn = Rows{(char*)grad_out->data, grad_out->s0 * size, grad_out->s1 * size, grad_out->s2 * size};
  if (grad_sum) a.dh = Rows{(char*)grad_sum->data, grad_sum->s0 * size, grad_sum->s1 * size, grad_sum->s2 * size};
  a.dx = (char*)dx;
  a.dbranch = (char*)dbranch;
  const bool ends = dgamma || dweight || dbias;
  RESS_REQUIRE(!ends || (workspace_bytes >= ress_layer_norm_bwd_workspace_size(c) && ((uintptr_t)workspace & 15) == 0 && (workspace || !a.rows)),
               "%s: the workspace is too small or not aligned", name);
  RESS_REQUIRE(!a.rows || (a.x.p && a.mean && a.rstd), "%s: null buffer", name);
  RESS_REQUIRE(a.branch.p || (!dbranch && !dgamma) || !a.rows, "%s: no branch", name);
  a.part = ends ? (float*)workspace : nullptr;
  const bool vec = a.C % 8 == 0 && aligned(a.x) && aligned(a.branch) && aligned(a.dn) && aligned(a.dh) && aligned(a.dx) &&
                   aligned(a.dbranch) && aligned(a.gamma) && aligned(a.weight) && aligned(a.part);
  int parts = 0;
  with_type(c->dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (a.rows)
      with_shape(a.C, vec, [&](auto tpr, auto k, auto v) {
        constexpr int T = decltype(tpr)::value, NT = ln_threads(T);
        parts = groups(a.rows, NT / T);
        hipLaunchKernelGGL((k_layer_norm_bwd<DT, T, decltype(k)::value, decltype(v)::value>), dim3(parts), dim3(NT), 0, stream, a);
      });
    if (ends) {
      const Ends e{{dweight, dbias, dgamma}, a.wide};
      hipLaunchKernelGGL((k_layer_norm_ends<DT>), dim3(cdiv(a.C, 64), 3), dim3(1024), 0, stream, a.part, parts, a.C, e);
    }
  });
  RESS_LAUNCHED("k_layer_norm_bwd");
  return 0;
}
