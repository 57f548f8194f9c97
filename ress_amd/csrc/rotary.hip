// Rotary positions: pairs of dims turned by a table of cosines and sines, and turned back for the backward pass.
//
//   (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin); the transpose has -sin
//
// Bound by the bytes of x and y (21,984 tokens of 16 + 16 heads of 64: 40 us, 4.5 TB/s; 16,384 of 32 + 8 heads of 128, half of their
// dims turned: 69 us, 4.9 TB/s), for few tokens by latency (32 tokens: 4 us). A thread takes 16 dims of a token (a unit: eight pairs, two 16-byte
// accesses each way) and goes through heads: positions are read, and cosines and sines fetched, once for all of them. The heads are cut into as many parts as
// give the card workgroups enough. Axes of other than 16 k dims, and operands that are not 16-byte aligned, go pair by pair.
#include "../../include/ress_hip.h"
#include "common.h"

namespace {

constexpr int ROT_BF16 = 1, ROT_F16 = 2;
constexpr int ROT_GROUPS = 2048;  // workgroups that fill the card (eight a CU)

struct Operand {
  const uint16_t* x;
  uint16_t* y;
  long long xb, xh, xt, yb, yh, yt;
  int H;
};
struct RotArgs {
  Operand o[2];
  int B, n, D, axes, d, interleaved;  // d: dims of an axis
  float sign;
  const long long* pos;
  long long pb, pt, pa;
  const float* table;
  int positions;
  int* status;
  int parts;  // of the heads, both operands' in one row
};

template <int DT>
__device__ __forceinline__ float widen(uint32_t bits) {
  if constexpr (DT == ROT_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  else return __uint_as_float(bits << 16);
}
template <int DT>
__device__ __forceinline__ uint32_t narrow(float x) {
  if constexpr (DT == ROT_F16) return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x);
  else return f32_to_bf16_bits(x);
}
template <int DT>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int u = 0; u < 8; ++u) x[u] = widen<DT>(u & 1 ? v[u >> 1] >> 16 : v[u >> 1] & 0xffffu);
}
template <int DT>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = narrow<DT>(x[2 * i]) | narrow<DT>(x[2 * i + 1]) << 16;
  return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ const float* table_row(const RotArgs& a, int b, int t, int axis) {
  long long p = a.pos[b * a.pb + t * a.pt + axis * a.pa];
  if (p < 0 || p >= a.positions) {
    atomicOr(a.status, 1);
    p = p < 0 ? 0 : a.positions - 1;
  }
  return a.table + p * a.d;  // d / 2 cosines, d / 2 sines
}

template <int DT, bool PAIRS>
__global__ __launch_bounds__(256) void k_rotate(RotArgs a) {
  const int units = a.D / 16;
  const unsigned i = blockIdx.x * 256 + threadIdx.x, token = i / units;  // fewer than 2^32 threads
  if (token >= (unsigned)a.B * (unsigned)a.n) return;
  const int u = (int)(i - token * units), b = (int)(token / (unsigned)a.n), t = (int)(token - (unsigned)b * a.n);
  const int turned = a.axes * a.d, d0 = 16 * u;
  const bool turn = d0 < turned;
  const int axis = turn ? d0 / a.d : 0, j = turn ? (d0 - axis * a.d) / 2 : 0;  // the unit's first pair
  float cs[8], sn[8];
  if (turn) {
    const float* row = table_row(a, b, t, axis) + j;
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const float4 c = *reinterpret_cast<const float4*>(row + e), s = *reinterpret_cast<const float4*>(row + a.d / 2 + e);
      cs[e] = c.x; cs[e + 1] = c.y; cs[e + 2] = c.z; cs[e + 3] = c.w;
      sn[e] = s.x * a.sign; sn[e + 1] = s.y * a.sign; sn[e + 2] = s.z * a.sign; sn[e + 3] = s.w * a.sign;
    }
  }
  // the unit's two pieces of 8 dims: neighbours, or those that turn together
  const int at0 = turn && !PAIRS ? axis * a.d + j : d0, at1 = turn && !PAIRS ? at0 + a.d / 2 : d0 + 8;
  const int heads = a.o[0].H + a.o[1].H, lo = (int)((long long)heads * blockIdx.y / a.parts),
            hi = (int)((long long)heads * (blockIdx.y + 1) / a.parts);
  for (int h = lo; h < hi; ++h) {
    const bool second = h >= a.o[0].H;
    const Operand& o = a.o[second];
    const int hh = second ? h - a.o[0].H : h;
    const uint16_t* x = o.x + b * o.xb + hh * o.xh + t * o.xt;
    uint16_t* y = o.y + b * o.yb + hh * o.yh + t * o.yt;
    uint4 w0 = *reinterpret_cast<const uint4*>(x + at0), w1 = *reinterpret_cast<const uint4*>(x + at1);
    if (turn) {
      float p[8], q[8];
      unpack8<DT>(w0, p);
      unpack8<DT>(w1, q);
      float r[8], s[8];
      if constexpr (PAIRS) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          r[2 * e] = fmaf(p[2 * e], cs[e], -(p[2 * e + 1] * sn[e]));
          r[2 * e + 1] = fmaf(p[2 * e + 1], cs[e], p[2 * e] * sn[e]);
          s[2 * e] = fmaf(q[2 * e], cs[4 + e], -(q[2 * e + 1] * sn[4 + e]));
          s[2 * e + 1] = fmaf(q[2 * e + 1], cs[4 + e], q[2 * e] * sn[4 + e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          r[e] = fmaf(p[e], cs[e], -(q[e] * sn[e]));
          s[e] = fmaf(q[e], cs[e], p[e] * sn[e]);
        }
      }
      w0 = pack8<DT>(r);
      w1 = pack8<DT>(s);
    }
    *reinterpret_cast<uint4*>(y + at0) = w0;
    *reinterpret_cast<uint4*>(y + at1) = w1;
  }
}

// a pair (or two dims that are copied) a thread
template <int DT>
__global__ __launch_bounds__(256) void k_rotate_any(RotArgs a) {
  const int units = a.D / 2;
  const unsigned i = blockIdx.x * 256 + threadIdx.x, token = i / units;  // fewer than 2^32 threads
  if (token >= (unsigned)a.B * (unsigned)a.n) return;
  const int u = (int)(i - token * units), b = (int)(token / (unsigned)a.n), t = (int)(token - (unsigned)b * a.n);
  const bool turn = 2 * u < a.axes * a.d;
  float c = 1.0f, s = 0.0f;
  int at0 = 2 * u, at1 = 2 * u + 1;
  if (turn) {
    const int axis = 2 * u / a.d, j = u - axis * (a.d / 2);
    const float* row = table_row(a, b, t, axis);
    c = row[j];
    s = row[a.d / 2 + j] * a.sign;
    if (!a.interleaved) {
      at0 = axis * a.d + j;
      at1 = at0 + a.d / 2;
    }
  }
  const int heads = a.o[0].H + a.o[1].H, lo = (int)((long long)heads * blockIdx.y / a.parts),
            hi = (int)((long long)heads * (blockIdx.y + 1) / a.parts);
  for (int h = lo; h < hi; ++h) {
    const bool second = h >= a.o[0].H;
    const Operand& o = a.o[second];
    const int hh = second ? h - a.o[0].H : h;
    const uint16_t* x = o.x + b * o.xb + hh * o.xh + t * o.xt;
    uint16_t* y = o.y + b * o.yb + hh * o.yh + t * o.yt;
    uint16_t w0 = x[at0], w1 = x[at1];
    if (turn) {
      const float p = widen<DT>(w0), q = widen<DT>(w1);
      w0 = (uint16_t)narrow<DT>(fmaf(p, c, -(q * s)));
      w1 = (uint16_t)narrow<DT>(fmaf(q, c, p * s));
    }
    y[at0] = w0;
    y[at1] = w1;
  }
}

bool vectors(const ress_strided& s) {
  return ((uintptr_t)s.data & 15) == 0 && ((s.sb | s.sh | s.st) & 7) == 0;
}

}  // namespace

RESS_API int ress_rotate(const ress_rotary* c, hipStream_t stream) {
  const char* name = "ress_rotate";
  RESS_REQUIRE(c, "%s: null arguments", name);
  RESS_REQUIRE(c->dtype == ROT_BF16 || c->dtype == ROT_F16, "%s: dtype code %d", name, c->dtype);
  RESS_REQUIRE(c->head_dim >= 2 && c->head_dim <= 256 && c->head_dim % 2 == 0, "%s: head_dim %d (even, up to 256)", name, c->head_dim);
  RESS_REQUIRE((c->axes == 1 || c->axes == 2) && c->rotary_dim >= 2 * c->axes && c->rotary_dim <= c->head_dim &&
                   c->rotary_dim % (2 * c->axes) == 0,
               "%s: %d dims to turn over %d axes, of %d", name, c->rotary_dim, c->axes, c->head_dim);
  RESS_REQUIRE(c->B >= 0 && c->n >= 0 && c->heads[0] >= 0 && c->heads[1] >= 0 && c->positions >= 1, "%s: bad geometry", name);
  if (!c->x[1].data) RESS_REQUIRE(c->heads[1] == 0, "%s: null buffer", name);
  const int heads = c->heads[0] + c->heads[1];
  if (!c->B || !c->n || !heads) return 0;
  RESS_REQUIRE(c->pos && c->table && c->status && ((uintptr_t)c->table & 15) == 0, "%s: null buffer or unaligned table", name);
  for (int i = 0; i < 2; ++i) RESS_REQUIRE(!c->heads[i] || (c->x[i].data && c->y[i].data), "%s: null buffer", name);
  RotArgs a{};
  const int d = c->rotary_dim / c->axes;
  bool vec = c->head_dim % 16 == 0 && d % 16 == 0;
  for (int i = 0; i < 2; ++i) {
    const ress_strided &x = c->x[i], &y = c->y[i];
    a.o[i] = Operand{(const uint16_t*)x.data, (uint16_t*)y.data, x.sb, x.sh, x.st, y.sb, y.sh, y.st, c->heads[i]};
    if (c->heads[i]) vec = vec && vectors(x) && vectors(y);
  }
  a.B = c->B;
  a.n = c->n;
  a.D = c->head_dim;
  a.axes = c->axes;
  a.d = d;
  a.interleaved = c->interleaved;
  a.sign = c->inverse ? -1.0f : 1.0f;
  a.pos = c->pos;
  a.pb = c->pos_sb;
  a.pt = c->pos_st;
  a.pa = c->pos_sa;
  a.table = c->table;
  a.positions = c->positions;
  a.status = c->status;
  const long long blocks = ((long long)c->B * c->n * (c->head_dim / (vec ? 16 : 2)) + 255) / 256;
  const long long parts = (ROT_GROUPS + blocks - 1) / blocks;
  a.parts = (int)(parts < heads ? parts : heads);
  RESS_REQUIRE(blocks * a.parts * 256 < 1ll << 32, "%s: 2^32 threads or more", name);
  const dim3 grid((unsigned)blocks, a.parts);
  if (c->dtype == ROT_BF16) {
    if (!vec) hipLaunchKernelGGL((k_rotate_any<ROT_BF16>), grid, dim3(256), 0, stream, a);
    else if (c->interleaved) hipLaunchKernelGGL((k_rotate<ROT_BF16, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((k_rotate<ROT_BF16, false>), grid, dim3(256), 0, stream, a);
  } else {
    if (!vec) hipLaunchKernelGGL((k_rotate_any<ROT_F16>), grid, dim3(256), 0, stream, a);
    else if (c->interleaved) hipLaunchKernelGGL((k_rotate<ROT_F16, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((k_rotate<ROT_F16, false>), grid, dim3(256), 0, stream, a);
  }
  RESS_LAUNCHED("k_rotate");
  return 0;
}
