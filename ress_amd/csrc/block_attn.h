// Parts of the attention kernels with a backward pass (block_attn.hip): operands, LDS tiles, lane layouts.
#pragma once
#include "common.h"

namespace {

constexpr int QB = 128, KB = 64, QS = 64;  // the map's query and key blocks; queries of a step of dK and dV
constexpr int BA_BF16 = 1, BA_F16 = 2;
constexpr float LOWEST = -0x1.fffffep127f;
// The running maximum moves when a score lies more than this above it (in log2): P stays below 2^8, and most steps need no
// pass over the accumulators.
constexpr float LAZY = 8.0f;
constexpr int VTOP_ROWS = 1024, DELTA_ROWS = 128;  // of a workgroup

typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

// A (B, heads, tokens, D) operand with unit-stride dims; strides in elements, tokens at least D apart
struct View {
  uint16_t* p;
  long long b, h, t;
  __device__ __forceinline__ uint16_t* at(int ib, int ih, int it) const { return p + ib * b + ih * h + it * t; }
};

struct AttnArgs {
  View q, k, v, o, go, dq, dk, dv;
  int B, Hq, Hk, G, Tq, Tk;  // G = Hq / Hk
  const int *q_lens, *k_lens;
  const uint8_t* map;        // bytes (b, h, query block, key block), not 0: kept
  long long mb, mh, mq, mk;
  int causal;
  float scale, scale2;       // scale2 = scale log2(e)
  uint16_t* rest;            // (B, Hq, Tq, D): what o's rounding took
  float *lse, *lse_b, *ndelta;  // (B, Hq, Tq); log2
  uint32_t* top;             // fp16: (B, Hk) largest |dO|, (B, Hk) largest |v|, as bits
  __device__ __forceinline__ int q_len(int b) const { return q_lens ? min(max(q_lens[b], 0), Tq) : Tq; }
  __device__ __forceinline__ int k_len(int b) const { return k_lens ? min(max(k_lens[b], 0), Tk) : Tk; }
  template <class I>
  __device__ __forceinline__ long long row_at(const I& it, int row) const {
    return ((long long)it.b * Hq + it.h) * Tq + row;
  }
};

// P's lift in the backward pass (log2): fp16 holds 2^-28 of a row's weight with all its bits
__device__ __forceinline__ constexpr float lift(int dt) { return dt == BA_F16 ? 14.0f : 0.0f; }
constexpr int tile_bytes(int D) { return KB * D * 2; }

// f(0), .., f(N - 1) with constant indexes, whatever the unroller decides: accumulator arrays stay in registers
template <int N, class F>
__device__ __forceinline__ void each(F f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}
__device__ __forceinline__ v16f zero16() {
  v16f z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.0f;
  return z;
}
template <int DT>
__device__ __forceinline__ v16f mfma(const uint4& a, const uint4& b, const v16f& c) {
  if constexpr (DT == BA_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const v2f x = {lo, hi};
  if constexpr (DT == BA_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, v2bf));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, v2h));
}
template <int DT>
__device__ __forceinline__ void pack16(const float (&e)[16], uint4 (&p)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    p[i] = make_uint4(pack2<DT>(e[8 * i], e[8 * i + 1]), pack2<DT>(e[8 * i + 2], e[8 * i + 3]),
                      pack2<DT>(e[8 * i + 4], e[8 * i + 5]), pack2<DT>(e[8 * i + 6], e[8 * i + 7]));
}
template <int DT>
__device__ __forceinline__ float unpack1(uint32_t w, int hi) {
  if constexpr (DT == BA_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(hi ? w >> 16 : w));
  else return hi ? bf16_hi(w) : bf16_lo(w);
}
template <int DT>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = unpack1<DT>(u[i >> 1], i & 1);
}
__device__ __forceinline__ float pair_max(float x) { return fmaxf(x, xor_lane_f<32>(x)); }
__device__ __forceinline__ float pair_sum(float x) { return x + xor_lane_f<32>(x); }

// Register r of a 32x32 result: row c_row(r) + 4 half
__device__ __forceinline__ constexpr int c_row(int r) { return (r & 3) + 8 * (r >> 2); }

// LDS tiles: 64 rows of D elements, a row's 16-byte chunks at chunk ^ f(row) (of 128 bytes),
// f(row) = 2 (row & 3) | (row >> 2 & 1): eight rows' reads of one chunk meet eight different 16-byte banks, and so do the
// four rows of two chunks that a 16-lane transposed read takes.
template <int D>
struct Lane {
  int wave, c32, half;
  int row_off[4];  // of chunk 2 s + half of row c32, s = 0..3 (s + 4: 128 bytes on)
  int col_off[2];  // of the lane's 8 bytes of a transposed read, dims 32 d.., d = 0, 1 (d + 2: 128 bytes on)
  __device__ __forceinline__ Lane() {
    const int l = threadIdx.x & 63, i = l & 15;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    c32 = l & 31;
    half = l >> 5;
    const int fr = (l & 3) << 1 | (l >> 2 & 1), fc = (i >> 2) << 1 | half;
#pragma unroll
    for (int s = 0; s < 4; ++s) row_off[s] = c32 * 2 * D + (((2 * s + half) ^ fr) << 4);
#pragma unroll
    for (int d = 0; d < 2; ++d)
      col_off[d] = (4 * half + (i >> 2)) * 2 * D + (((4 * d + 2 * (l >> 4 & 1) + (i >> 1 & 1)) ^ fc) << 4) + 8 * (i & 1);
  }
};

// rows row0..row0+31 of the tile (A) times the lane's 16-bit operand (B), over D dims
template <int DT, int D>
__device__ __forceinline__ v16f rows_times(const uint8_t* tile, int row0, const Lane<D>& ln, const uint4 (&b)[D / 16],
                                           v16f acc) {
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    const uint4 x = *reinterpret_cast<const uint4*>(tile + row0 * 2 * D + ln.row_off[s & 3] + (s >> 2) * 128);
    acc = mfma<DT>(x, b[s], acc);
  }
  return acc;
}
__device__ __forceinline__ uint2 read_tr(const uint8_t* p) {
  typedef __attribute__((address_space(3))) v4s* lds_v4s;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(void*)const_cast<uint8_t*>(p)));
}
// dims 32 d.. of rows row0..row0+31, transposed (A), times b (B), over the 32 rows in the order of a result's registers
template <int DT, int D>
__device__ __forceinline__ v16f columns_times(const uint8_t* tile, int row0, int d, const Lane<D>& ln, const uint4 (&b)[2],
                                              v16f acc) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint8_t* p = tile + (row0 + 16 * s) * 2 * D + ln.col_off[d & 1] + (d >> 1) * 128;
    const uint2 lo = read_tr(p), hi = read_tr(p + 8 * 2 * D);
    acc = mfma<DT>(make_uint4(lo.x, lo.y, hi.x, hi.y), b[s], acc);
  }
  return acc;
}
// The lane's B operand of a row: dims 16 s + 8 half ..
template <int D>
__device__ __forceinline__ void load_row(const View& x, int b, int h, int row, bool live, int half, uint4 (&f)[D / 16]) {
#pragma unroll
  for (int s = 0; s < D / 16; ++s)
    f[s] = live ? *reinterpret_cast<const uint4*>(x.at(b, h, row) + 16 * s + 8 * half) : make_uint4(0, 0, 0, 0);
}

// ---- LDS-DMA ------------------------------------------------------------------
// A buffer of `bytes` bytes at `base` (wave-uniform): reads past its end give zero.
__device__ __forceinline__ v4i descriptor(const void* base, unsigned bytes) {
  const unsigned long long p = (unsigned long long)base;
  return v4i{__builtin_amdgcn_readfirstlane((int)(unsigned)p), __builtin_amdgcn_readfirstlane((int)(unsigned)(p >> 32)),
             __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return __builtin_amdgcn_readfirstlane((unsigned)(unsigned long long)(__attribute__((address_space(3))) void*)const_cast<void*>(p));
}
// 16 (4) bytes a lane from the buffer at off into LDS at lds + 16 (4) lane. As assembly, because the compiler waits for every
// DMA in flight before an LDS read of a buffer that one fills; no output register, m0 set in the same block.
__device__ __forceinline__ void dma16(const v4i& rsrc, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(lds), "v"(off), "s"(rsrc)
               : "memory", "m0");
}
__device__ __forceinline__ void dma4(const v4i& rsrc, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" : : "s"(lds), "v"(off), "s"(rsrc)
               : "memory", "m0");
}
// every DMA of the wave has landed and its LDS reads are done, then the workgroup's
__device__ __forceinline__ void step_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Tiles of 64 rows of a (sequence, head), filled by the workgroup's waves: 1 KB a DMA. Rows past `len` are zero.
template <int D>
struct Stream {
  static constexpr int RPD = 512 / D, ND = 64 / RPD;  // rows of a DMA, DMAs of a tile
  const uint16_t* base;
  unsigned stride, lane_off;  // bytes
  int nw;
  __device__ __forceinline__ Stream(const View& x, const uint16_t* head, const Lane<D>& ln, int nw_) : base(head), nw(nw_) {
    const int l = threadIdx.x & 63, r = l / (D / 8), slot = l % (D / 8);
    const int row = D == 64 ? r : 4 * (ln.wave & 1) + r;  // & 7; a wave's DMAs are all even or all odd
    stride = (unsigned)(2 * x.t);
    lane_off = r * stride + ((slot ^ ((row & 3) << 1 | (row >> 2 & 1))) << 4);
  }
  __device__ __forceinline__ void fetch(const uint8_t* lds, int row0, int len, int w) const {
    const int rows = min(64, len - row0);
    const v4i rs = descriptor(reinterpret_cast<const char*>(base) + (long long)row0 * stride, (rows - 1) * stride + 2 * D);
    const unsigned at = lds_address(lds);
    for (int n = w; n < ND; n += nw) dma16(rs, lane_off + n * RPD * stride, at + n * 1024);
  }
};
// 64 values, one for each row of a tile (zero past `left`)
__device__ __forceinline__ void fetch_row_values(const float* src, int left, const uint8_t* lds) {
  dma4(descriptor(src, 4 * min(64, left)), 4 * (threadIdx.x & 63), lds_address(lds));
}
template <int D>
__device__ __forceinline__ v16f row_values(const uint8_t* lds, int row0, const Lane<D>& ln) {
  v16f x;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const v4f y = *reinterpret_cast<const v4f*>(lds + 4 * (row0 + 8 * g + 4 * ln.half));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[4 * g + i] = y[i];
  }
  return x;
}

// ---- work -----------------------------------------------------------------------
// A workgroup's tile. An XCD (workgroup i runs on XCD i % 8) takes consecutive tiles, so that a head's keys and values, or
// its queries, are read through few L2s. Causal: query tiles from the last one on, which see most.
struct Item {
  int b, h, tile;
  __device__ __forceinline__ bool place(const AttnArgs& a, int heads, int tiles) {
    const long long total = (long long)a.B * heads * tiles, per = (total + 7) / 8;
    const long long lin = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per || lin >= total) return false;
    const int bh = (int)(lin / tiles);
    tile = (int)(lin % tiles);
    b = bh / heads;
    h = bh % heads;
    return true;
  }
  __device__ __forceinline__ bool query_tile(const AttnArgs& a) {
    const int tiles = cdiv(a.Tq, QB);
    if (!place(a, a.Hq, tiles)) return false;
    if (a.causal) tile = tiles - 1 - tile;
    return true;
  }
  __device__ __forceinline__ bool key_tile(const AttnArgs& a, int keys) { return place(a, a.Hk, cdiv(a.Tk, keys)); }
};
struct Head {
  int b, h, klen;
  __device__ __forceinline__ Head(const AttnArgs& a, int b_, int h_) : b(b_), h(h_), klen(a.k_len(b_)) {}
  __device__ __forceinline__ const uint16_t* kbase(const View& x) const { return x.at(b, h, 0); }
};

// The kept entries of a line of the map as bits in LDS
struct Bits {
  const uint32_t* bits;
  int n;
  __device__ __forceinline__ void fill(const uint8_t* line, long long step, int n_, uint32_t* to) {
    bits = to;
    n = n_;
    const int lane = threadIdx.x & 63;
    for (int j = (threadIdx.x >> 6) * 64; j < n; j += blockDim.x) {
      const unsigned long long m = __ballot(j + lane < n && line[(long long)(j + lane) * step] != 0);
      if (lane == 0) {
        to[j >> 5] = (uint32_t)m;
        to[(j >> 5) + 1] = (uint32_t)(m >> 32);
      }
    }
    __syncthreads();
  }
  // the first kept entry from j on, or -1
  __device__ __forceinline__ int from(int j) const {
    while (j < n) {
      const uint32_t w = (uint32_t)__builtin_amdgcn_readfirstlane((int)bits[j >> 5]) >> (j & 31);
      if (w) return j + __builtin_ctz(w);
      j = (j | 31) + 1;
    }
    return -1;
  }
};
// The key blocks 0..n-1 that a query tile goes through
template <bool MAP>
struct Walk {
  Bits bits;
  int n;
  __device__ __forceinline__ Walk(const AttnArgs& a, const Item& it, int n_, uint32_t* lds) : n(n_) {
    if constexpr (MAP) bits.fill(a.map + it.b * a.mb + it.h * a.mh + it.tile * a.mq, a.mk, n, lds);
  }
  __device__ __forceinline__ int first() const { return next(-1); }
  __device__ __forceinline__ int next(int i) const {
    if constexpr (MAP) return bits.from(i + 1);
    else return i + 1 < n ? i + 1 : -1;
  }
};
// The steps of 64 queries from `start` to n-1 that key block `col` goes through
template <bool MAP>
struct WalkColumn {
  Bits bits;
  int start, n;
  __device__ __forceinline__ WalkColumn(const AttnArgs& a, int b, int h, int col, int start_, int n_, uint32_t* lds, bool again)
      : start(start_), n(n_) {
    if (again) __syncthreads();  // the head before is done with the tiles and the bits
    if constexpr (MAP) bits.fill(a.map + b * a.mb + h * a.mh + col * a.mk, a.mq, cdiv(n, QB / QS), lds);
  }
  __device__ __forceinline__ int first() const { return from(start); }
  __device__ __forceinline__ int next(int i) const { return from(i + 1); }
  __device__ __forceinline__ int from(int st) const {
    if (st >= n) return -1;
    if constexpr (MAP) {
      const int q = bits.from(st / (QB / QS));
      if (q < 0) return -1;
      st = max(st, q * (QB / QS));
    }
    return st;
  }
};
// Every step: its tile has landed, the next one's DMAs go out into the other buffer (which all waves have left), compute.
template <class W, class F, class C>
__device__ __forceinline__ void run_steps(const W& walk, F fetch, C compute) {
  int cur = walk.first(), buf = 0;
  if (cur < 0) return;
  fetch(0, cur);
  while (cur >= 0) {
    const int nxt = walk.next(cur);
    step_barrier();
    if (nxt >= 0) fetch(buf ^ 1, nxt);
    compute(buf, cur);
    cur = nxt;
    buf ^= 1;
  }
}

// ---- results --------------------------------------------------------------------
template <int DT, int D>
__device__ __forceinline__ void store_grad(const View& x, int b, int h, int row, int half, const v16f (&acc)[D / 32], float by,
                                           bool live) {
  uint16_t* to = x.at(b, h, row) + 4 * half;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint2 y = make_uint2(pack2<DT>(acc[d][4 * g] * by, acc[d][4 * g + 1] * by),
                           pack2<DT>(acc[d][4 * g + 2] * by, acc[d][4 * g + 3] * by));
      if (!live) y = make_uint2(0, 0);
      *reinterpret_cast<uint2*>(to + 32 * d + 8 * g) = y;
    }
}
template <int DT, int D>
__device__ __forceinline__ void store_out(const AttnArgs& a, const Item& it, int row, int half, const v16f (&o)[D / 32], float by,
                                          bool live) {
  uint16_t* to = a.o.at(it.b, it.h, row) + 4 * half;
  uint16_t* rest = a.rest ? a.rest + a.row_at(it, row) * D + 4 * half : nullptr;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = live ? o[d][4 * g + i] * by : 0.0f;
      const uint2 y = make_uint2(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]));
      *reinterpret_cast<uint2*>(to + 32 * d + 8 * g) = y;
      if (rest) {
        const uint2 z = make_uint2(pack2<DT>(x[0] - unpack1<DT>(y.x, 0), x[1] - unpack1<DT>(y.x, 1)),
                                   pack2<DT>(x[2] - unpack1<DT>(y.y, 0), x[3] - unpack1<DT>(y.y, 1)));
        *reinterpret_cast<uint2*>(rest + 32 * d + 8 * g) = z;
      }
    }
}

}  // namespace
