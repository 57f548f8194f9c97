// Parts of the attention kernels with a backward pass (block_attn.hip): operands, LDS tiles, lane layouts.
#pragma once
#include "common.h"

namespace {

constexpr int QB = 128, KB = 64;  // the map's query and key blocks
// Rows of a streamed tile: 8 KB of an operand, in tiles of 32 for the matrix cores
constexpr int step_rows(int D) { return 4096 / D; }
constexpr int BA_BF16 = 1, BA_F16 = 2;
constexpr float LOWEST = -0x1.fffffep127f;
// The running maximum moves when a score lies more than this above it (in log2): P stays below 2^8, and most steps need no
// pass over the accumulators.
constexpr float LAZY = 8.0f;
constexpr int DELTA_ROWS = 128;  // of a workgroup

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
  // A tile's steps cut into parts (where the tiles are few), a workgroup each: grid.y. Parts of rows (o or dq, and lse) or of
  // keys (dk, dv): [part][rows][D], [part][rows]
  int parts;
  float *part, *part2;
  __device__ __forceinline__ int q_len(int b) const { return q_lens ? min(max(q_lens[b], 0), Tq) : Tq; }
  __device__ __forceinline__ int k_len(int b) const { return k_lens ? min(max(k_lens[b], 0), Tk) : Tk; }
  template <class I>
  __device__ __forceinline__ long long row_at(const I& it, int row) const {
    return ((long long)it.b * Hq + it.h) * Tq + row;
  }
};

// P's lift in the backward pass (log2): fp16 holds 2^-28 of a row's weight with all its bits
__device__ __forceinline__ constexpr float lift(int dt) { return dt == BA_F16 ? 14.0f : 0.0f; }

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
// What rounding took of e, rounded in its turn
template <int DT>
__device__ __forceinline__ void pack_rest(const float (&e)[16], const uint4 (&p)[2], uint4 (&rest)[2]) {
  float x[16];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float y[8];
    unpack8<DT>(p[i], y);
#pragma unroll
    for (int u = 0; u < 8; ++u) x[8 * i + u] = e[8 * i + u] - y[u];
  }
  pack16<DT>(x, rest);
}
__device__ __forceinline__ float sum16(const float (&e)[16]) {
  float s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = (e[i] + e[4 + i]) + (e[8 + i] + e[12 + i]);
  return (s[0] + s[1]) + (s[2] + s[3]);
}
__device__ __forceinline__ float pair_max(float x) { return fmaxf(x, xor_lane_f<32>(x)); }
__device__ __forceinline__ float pair_sum(float x) { return x + xor_lane_f<32>(x); }

// Register r of a 32x32 result: row c_row(r) + 4 half
__device__ __forceinline__ constexpr int c_row(int r) { return (r & 3) + 8 * (r >> 2); }

// LDS tiles: rows of D elements, a row's 16-byte chunks at chunk ^ f(row). f takes the row's bits 1, 2, 3 (D = 128: 0 to 3) from
// the chunk's highest bit down: 16 rows' reads of one chunk meet 16 different places of the 256 bytes that the banks
// hold, and so do the four rows of four chunks that 32 lanes of a transposed read take. (With f of three bits alone, row reads
// met a bank twice: 40% of the LDS' cycles.)
template <int D>
__device__ __forceinline__ int swizzle(int row) {
  const int f = (row & 2) << 1 | (row >> 1 & 2) | (row >> 3 & 1);
  return D == 128 ? f | (row & 1) << 3 : f;
}
template <int D>
struct Lane {
  int wave, c32, half;
  int row_at;  // of chunk `half` of row c32: chunk 2 s + half is at row_at ^ 32 s
  int col_at;  // of the lane's 8 bytes of a transposed read of dims 0.. of rows 0..: dims 32 d.. at col_at ^ 64 d, rows 8.. at
               // (col_at ^ 16) + 8 rows
  __device__ __forceinline__ Lane() {
    const int l = threadIdx.x & 63, i = l & 15;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    c32 = l & 31;
    half = l >> 5;
    row_at = c32 * 2 * D + ((half ^ swizzle<D>(c32)) << 4);
    const int r = 4 * half + (i >> 2);
    col_at = r * 2 * D + (((2 * (l >> 4 & 1) + (i >> 1 & 1)) ^ swizzle<D>(r)) << 4) + 8 * (i & 1);
  }
  // The same, opaque to the compiler: the places derived from it are formed where they are used and not held in
  // registers through a loop that has none to spare.
  __device__ __forceinline__ Lane anew() const {
    Lane x = *this;
    asm volatile("" : "+v"(x.row_at), "+v"(x.col_at));
    return x;
  }
};

// rows row0..row0+31 of the tile (A) times the lane's 16-bit operand (B), over D dims
template <int DT, int D>
__device__ __forceinline__ v16f rows_times(const uint8_t* tile, int row0, const Lane<D>& ln, const uint4 (&b)[D / 16],
                                           v16f acc) {
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    const uint4 x = *reinterpret_cast<const uint4*>(tile + row0 * 2 * D + (ln.row_at ^ 32 * s));
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
    const uint8_t* p = tile + (row0 + 16 * s) * 2 * D;
    const uint2 lo = read_tr(p + (ln.col_at ^ 64 * d)), hi = read_tr(p + 8 * 2 * D + (ln.col_at ^ 64 * d ^ 16));
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
// all but the wave's newest N DMAs have landed and its LDS reads are done, then the workgroup's
template <int N>
__device__ __forceinline__ void step_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Tiles of ROWS rows of a (sequence, head), filled by the workgroup's NW waves: 1 KB a DMA. Rows past `len` are zero.
template <int D, int NW, int ROWS = step_rows(D)>
struct Stream {
  static constexpr int RPD = 512 / D, DMAS = ROWS / RPD / NW;  // rows of a DMA, DMAs of a wave
  static_assert(NW * RPD % 16 == 0, "a wave's DMAs go to rows of one swizzle");
  const uint16_t* base;
  unsigned stride, off;  // bytes
  __device__ __forceinline__ Stream(const View& x, const uint16_t* head, const Lane<D>& ln) : base(head) {
    const int l = threadIdx.x & 63, slot = l % (D / 8), row = ln.wave * RPD + l / (D / 8);
    stride = (unsigned)(2 * x.t);
    off = row * stride + ((slot ^ swizzle<D>(row)) << 4);
  }
  // lds: the tile's address
  __device__ __forceinline__ void fetch(unsigned lds, int row0, int len, int w) const {
    const int rows = min(ROWS, len - row0);
    const v4i rs = descriptor(reinterpret_cast<const char*>(base) + (long long)row0 * stride, (rows - 1) * stride + 2 * D);
    unsigned at = off;
    asm volatile("" : "+v"(at));  // sums formed here, not held in registers through the loop
    // the rows go into the offset that is checked, not into the scalar one
#pragma unroll
    for (int n = 0; n < DMAS; ++n) dma16(rs, at + n * NW * RPD * stride, lds + (n * NW + w) * 1024);
  }
};
// 64 values (zero past `left`)
__device__ __forceinline__ void fetch_row_values(const float* src, int left, unsigned lds) {
  dma4(descriptor(src, 4 * min(64, left)), 4 * (threadIdx.x & 63), lds);
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
// A workgroup's tile. Workgroup i runs on XCD i % 8: whole heads go to the XCDs in turn (their lengths differ by sequence, and
// a head's tiles read the same keys), what eight do not divide in eight runs of tiles. Causal: the tiles that see most first, and
// the heads in an order that turns from tile to tile where a sequence has not four of them an XCD: an XCD's workgroups go to its four
// shader engines in turn, and an engine had all tiles of the same sequences (four of 549 to 2,048 tokens, eight key heads of
// 128: dK and dV 278 us for 243).
struct Item {
  int b, h, tile;
  __device__ __forceinline__ bool place(const AttnArgs& a, int heads, int tiles, bool by_tile) {
    const int all = a.B * heads, x = blockIdx.x & 7, i = blockIdx.x >> 3, even = all / 8;
    int bh;
    if (i < even * tiles) {
      tile = by_tile ? i / even : i % tiles;
      const int turn = heads % 32 == 0 ? 0 : even % 4 == 0 ? tile : even % 2 == 0 ? tile / 2 : 0;
      bh = (by_tile ? (i % even + turn) % even : i / tiles) * 8 + x;
    } else {
      const int left = (all - 8 * even) * tiles, per = (left + 7) / 8, j = i - even * tiles;
      const int lin = x * per + j;
      if (j >= per || lin >= left) return false;
      bh = 8 * even + lin / tiles;
      tile = lin % tiles;
    }
    // divisions go through vector registers; what follows from these must not
    tile = __builtin_amdgcn_readfirstlane(tile);
    bh = __builtin_amdgcn_readfirstlane(bh);
    b = __builtin_amdgcn_readfirstlane(bh / heads);
    h = bh - b * heads;
    return true;
  }
  __device__ __forceinline__ bool query_tile(const AttnArgs& a) {
    const int tiles = cdiv(a.Tq, QB);
    if (!place(a, a.Hq, tiles, a.causal)) return false;
    if (a.causal) tile = tiles - 1 - tile;
    return true;
  }
  __device__ __forceinline__ bool key_tile(const AttnArgs& a, int keys) {
    return place(a, a.Hk, cdiv(a.Tk, keys), a.causal);
  }
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
// The steps start..n-1 that a workgroup goes through; with a map, PER of them to an entry of its line
template <bool MAP, int PER>
struct Walk {
  Bits bits;
  int start, n;
  // line[i step]: the entry of steps PER i..; again: the walk before may still be in use
  __device__ __forceinline__ Walk(const uint8_t* line, long long step, int start_, int n_, uint32_t* lds, bool again)
      : start(start_), n(n_) {
    if (again) __syncthreads();
    if constexpr (MAP) bits.fill(line, step, cdiv(n, PER), lds);
  }
  __device__ __forceinline__ int first() const { return from(start); }
  __device__ __forceinline__ int next(int i) const { return from(i + 1); }
  __device__ __forceinline__ int from(int st) const {
    if (st >= n) return -1;
    if constexpr (MAP) {
      const int e = bits.from(st / PER);
      if (e < 0) return -1;
      st = max(st, e * PER);
    }
    return st;
  }
};
// Steps through NS stages of LDS, the DMAs (N a wave and stage) NS - 1 steps ahead: the step's stage has landed in every wave,
// the DMAs of a later step go out into the stage that all waves have left, compute. The steps for which `early` holds come first
// and are a loop of their own, with a body of their own: in one loop with two bodies the accumulators did not keep
// their registers.
template <int NS, int N, class W, class F, class E, class A, class B>
__device__ __forceinline__ void run_steps(const W& walk, F fetch, E early, A compute_early, B compute_late) {
  static_assert(NS == 2 || NS == 3, "");
  int cur = walk.first(), stage = 0;
  if (cur < 0) return;
  fetch(0, cur);
  int nxt = walk.next(cur);
  if constexpr (NS == 3) {
    if (nxt >= 0) fetch(1, nxt);
  }
  auto step = [&](auto compute) {
    if constexpr (NS == 3) {
      if (nxt >= 0) step_barrier<N>();
      else step_barrier<0>();
      const int after = nxt >= 0 ? walk.next(nxt) : -1;
      if (after >= 0) fetch(stage == 0 ? 2 : stage - 1, after);
      compute(stage, cur);
      cur = nxt;
      nxt = after;
      stage = stage == 2 ? 0 : stage + 1;
    } else {
      step_barrier<0>();
      if (nxt >= 0) fetch(stage ^ 1, nxt);
      compute(stage, cur);
      cur = nxt;
      if (nxt >= 0) nxt = walk.next(nxt);
      stage ^= 1;
    }
  };
  while (cur >= 0 && early(cur)) step(compute_early);
  while (cur >= 0) step(compute_late);
}

// Part p of the steps 0..n-1
__device__ __forceinline__ int part_of(int n, int p, int parts) { return (int)((long long)n * p / parts); }

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
// a part's sums in fp32, rows of D
template <int D>
__device__ __forceinline__ void store_part(float* row, int half, const v16f (&acc)[D / 32], float by, bool live) {
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      v4f y;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = live ? acc[d][4 * g + i] * by : 0.0f;
      *reinterpret_cast<v4f*>(row + 32 * d + 8 * g + 4 * half) = y;
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
