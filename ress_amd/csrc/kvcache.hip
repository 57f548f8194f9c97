// Writing and reading back the paged 8-bit key/value cache (layout: kvcache.h).
//
// Rotation. For an axis of d dims (d = D / axes, dims [a d, (a+1) d)) at position p, with cos and sin of
// p * base^(-2i/d) from a table: r[i] = x[i] c_i - x[i + d/2] s_i, r[i + d/2] = x[i + d/2] c_i + x[i] s_i,
// i < d/2, each product and sum rounded in fp32 and the result once to 16 bits. One axis is the usual
// rotary embedding of a token's index, two are the rows and columns of a patch grid.
//
// Codes. A page that is full has for each head and for keys and values apart a = max |x| over its 64 D
// elements, code = rne(x * min(M / a, FLT_MAX)) and scale = a * fl(1 / M), M = 127 (int8) or 448 (e4m3);
// a = 0 gives scale 0. With an element that is not finite the codes are 0 and the scale NaN, so that
// every query that sees a token of the page gets NaN and no other is touched. A page that is not full stays
// in 16 bits and is quantised when its last token comes: what the cache holds does not hang on how the
// tokens were split over calls, and no code is ever rounded twice.
#include "kvcache.h"

namespace {

constexpr int THREADS = 256;
constexpr int QH = 4;  // query heads a workgroup rotates together

struct AppendArgs {
  ress_kv_cache c;
  const uint16_t *k, *v, *q;
  long long skb, skh, skt, svb, svh, svt, sqb, sqh, sqt;
  const long long* pos;   // (B, n, axes) or null
  const float* rope;      // (positions, 2, D / 2 / axes)
  int positions, axes;
  int B, Hq, n;
  const int *slots, *new_lens;
  uint16_t* q_out;        // (B, Hq, n, D)
  int pages;              // pages a sequence's new tokens can touch
  bool vec;               // k, v, q and their strides are 16-byte aligned
};

__device__ __forceinline__ int new_tokens(const int* new_lens, int b, int n) {
  return new_lens ? min(max(new_lens[b], 0), n) : n;
}

// The chunk pair of a row that a lane owns: dims x1.. and x2.., 8 each, rotation partners of each other.
template <int D>
struct Pair {
  int x1, x2, f, axis;  // first dims, first frequency, axis
  __device__ __forceinline__ Pair(int lane, int axes) {
    const int half = D / 2 / axes, per = half / 8;  // chunk pairs per axis
    axis = lane / per;
    f = (lane % per) * 8;
    x1 = axis * 2 * half + f;
    x2 = x1 + half;
  }
};

template <int DT>
__device__ __forceinline__ void rotate(uint4& a, uint4& b, const float* __restrict__ cs, const float* __restrict__ sn) {
  uint16_t ra[8], rb[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = Elem<DT>::get(elem8(a, i)), y = Elem<DT>::get(elem8(b, i));
    const float c = cs[i], s = sn[i];
    const float xc = x * c, ys = y * s, yc = y * c, xs = x * s;
    ra[i] = Elem<DT>::put(xc - ys);
    rb[i] = Elem<DT>::put(yc + xs);
  }
  a = pack8(ra);
  b = pack8(rb);
}

// The table row of a token, its positions clamped into the table (`out` set, for the status word: an atomic here would
// keep the loads behind it from being issued early).
__device__ __forceinline__ const float* rope_row(const AppendArgs& a, int b, int i, int axis, int half, bool& out) {
  const long long p = a.pos[((long long)b * a.n + i) * a.axes + axis];
  out = out || p < 0 || p >= a.positions;
  const long long pc = p < 0 ? 0 : p >= a.positions ? a.positions - 1 : p;
  return a.rope + pc * 2 * half;
}

// The largest |x| bits (the sign off) of a uint4 of 16-bit elements
__device__ __forceinline__ uint32_t top_bits(const uint4& v, uint32_t m) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
  return m;
}

// One workgroup handles, for a (sequence, head): workgroup 0 the page the sequence ends in and, after it,
// the new last page; the others a page each that the call fills. The unfinished page's 16-bit tokens are
// read and rewritten by workgroup 0 alone, in that order. The queries' workgroups follow in the same launch.
//
// A page's tokens stay in registers between its maximum and its codes, so they are read once; a head's values are
// transposed through LDS, in rows of 17 words, and leave as whole lines. Bound by memory where there is much to append
// (8 sequences of up to 1,000 tokens, 24 heads of 64: 30 us for 110 MB, 3.6 TB/s), else by the chain length -> tokens ->
// maximum -> codes -> length (1,374 tokens of 16 heads, 10 us for 14 MB; a token each of 32 sequences, 8 us): with
// the first tokens on their way before the length is known and each sequence's counter on a line of its own it took
// 66 -> 50 us of the first, its reading back included.
template <int DT, int CODES, int D>
__global__ __launch_bounds__(THREADS) void k_kv_append(AppendArgs a, int kv_groups) {
  constexpr int LPR = D / 16;               // lanes per row
  constexpr int ROWS = THREADS / LPR;       // rows at a time
  constexpr int IT = KV_PAGE / ROWS;        // passes over a page
  constexpr int VROW = KV_PAGE + 4;         // LDS row of transposed codes: 17 words, stores spread over the banks
  __shared__ __align__(16) uint8_t vt[D * VROW];
  __shared__ uint32_t red[2][THREADS / 64];
  const int t = threadIdx.x, H = a.c.kv_heads;
  const int half = D / 2 / a.axes;
  const Pair<D> pr(t % LPR, a.axes);

  bool outside = false;
  if ((int)blockIdx.x >= kv_groups) {  // the queries: ROWS tokens of QH heads a workgroup, the table read once for them
    const int hgs = cdiv(a.Hq, QH), tgs = cdiv(a.n, ROWS);
    int g = blockIdx.x - kv_groups;
    const int tg = g % tgs, hg = g / tgs % hgs, b = g / tgs / hgs, i = tg * ROWS + t / LPR, h0 = hg * QH;
    if (i >= a.n) return;
    const bool there = i < new_tokens(a.new_lens, b, a.n);
    uint4 x[QH], y[QH];
#pragma unroll
    for (int j = 0; j < QH; ++j) {
      x[j] = y[j] = make_uint4(0, 0, 0, 0);
      if (there && h0 + j < a.Hq) {
        const uint16_t* src = a.q + b * a.sqb + (h0 + j) * a.sqh + i * a.sqt;
        x[j] = ld8(src + pr.x1, a.vec);
        y[j] = ld8(src + pr.x2, a.vec);
      }
    }
    float cs[8], sn[8];
    if (there) {
      const float* tb = rope_row(a, b, i, pr.axis, half, outside) + pr.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cs[j] = tb[j];
        sn[j] = tb[half + j];
      }
    }
#pragma unroll
    for (int j = 0; j < QH; ++j) {
      if (h0 + j >= a.Hq) break;
      if (there) rotate<DT>(x[j], y[j], cs, sn);
      uint16_t* dst = a.q_out + (((long long)b * a.Hq + h0 + j) * a.n + i) * D;
      *reinterpret_cast<uint4*>(dst + pr.x1) = x[j];
      *reinterpret_cast<uint4*>(dst + pr.x2) = y[j];
    }
    if (outside) atomicOr(a.c.status, KV_ST_POS);
    return;
  }

  const int part = blockIdx.x % a.pages, h = blockIdx.x / a.pages % H, b = blockIdx.x / a.pages / H;
  bool there;
  const int slot = slot_of(a.c, a.slots, b, there);
  if (!there) {
    if (t == 0 && part == 0 && h == 0) atomicOr(a.c.status, KV_ST_SLOT);
    return;
  }

  const int held = a.c.held[slot], cap = held * KV_PAGE, fresh = new_tokens(a.new_lens, b, a.n);
  const int len = held_tokens(a.c.lens[slot], held);
  const long long tail = ((long long)slot * H + h) * KV_PAGE * D;
  uint16_t* tail_k = reinterpret_cast<uint16_t*>(a.c.tail_k) + tail;
  uint16_t* tail_v = reinterpret_cast<uint16_t*>(a.c.tail_v) + tail;
  float* tail_top = a.c.tail_top + (long long)slot * H + h;
  const float top0 = part == 0 ? *tail_top : 0.0f;

  // new token i of the sequence, this lane's dims, rotated
  auto token = [&](int i, uint4& kx, uint4& ky, uint4& vx, uint4& vy) {
    const uint16_t* ks = a.k + b * a.skb + h * a.skh + i * a.skt;
    const uint16_t* vs = a.v + b * a.svb + h * a.svh + i * a.svt;
    kx = ld8(ks + pr.x1, a.vec);
    ky = ld8(ks + pr.x2, a.vec);
    vx = ld8(vs + pr.x1, a.vec);
    vy = ld8(vs + pr.x2, a.vec);
    if (a.pos) {
      const float* tb = rope_row(a, b, i, pr.axis, half, outside) + pr.f;
      rotate<DT>(kx, ky, tb, tb + half);
    }
  };
  // The first tokens (all of them in a decoding step) on their way before the sequence's length is known, for the
  // case that they fill no page.
  const int mine = t / LPR;
  uint4 kx0, ky0, vx0, vy0;
  kx0 = ky0 = vx0 = vy0 = make_uint4(0, 0, 0, 0);
  if (a.n < KV_PAGE && part == 0 && mine < fresh) token(mine, kx0, ky0, vx0, vy0);
  const int end = len + min(fresh, max(cap - len, 0));
  const int p0 = len / KV_PAGE, p1 = end / KV_PAGE;  // pages p0..p1-1 get full, p1 stays open
  if (t == 0 && part == 0 && h == 0 && end < len + (long long)fresh) atomicOr(a.c.status, KV_ST_FULL);

  auto page = [&](int pg, bool full) {
    uint4 kx[IT], ky[IT], vx[IT], vy[IT];
    uint32_t ktop = 0, vtop = 0;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int r = it * ROWS + t / LPR, tok = pg * KV_PAGE + r;
      kx[it] = ky[it] = vx[it] = vy[it] = make_uint4(0, 0, 0, 0);
      if (tok < len) {  // held in 16 bits (only the page the sequence ended in has such)
        if (full) {
          kx[it] = *reinterpret_cast<const uint4*>(tail_k + r * D + pr.x1);
          ky[it] = *reinterpret_cast<const uint4*>(tail_k + r * D + pr.x2);
          uint16_t e[8], f[8];
          const int pl = v_place(r);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            e[i] = tail_v[(pr.x1 + i) * KV_PAGE + pl];
            f[i] = tail_v[(pr.x2 + i) * KV_PAGE + pl];
          }
          vx[it] = pack8(e);
          vy[it] = pack8(f);
        }
      } else if (tok < end) {
        token(tok - len, kx[it], ky[it], vx[it], vy[it]);
      }
      ktop = top_bits(ky[it], top_bits(kx[it], ktop));
      vtop = top_bits(vy[it], top_bits(vx[it], vtop));
    }
    __syncthreads();  // the last use of red, vt and of the tail by this workgroup's other call
    ktop = wave_max_u32(ktop);
    vtop = wave_max_u32(vtop);
    if ((t & 63) == 0) {
      red[0][t >> 6] = ktop;
      red[1][t >> 6] = vtop;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      ktop = max(ktop, red[0][w]);
      vtop = max(vtop, red[1][w]);
    }
    const float nan = __uint_as_float(0x7fc00000u);
    const bool kbad = ktop >= Elem<DT>::INF, vbad = vtop >= Elem<DT>::INF;
    const float kt = Elem<DT>::get((uint16_t)ktop), vt_ = Elem<DT>::get((uint16_t)vtop);

    if (!full) {
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const int r = it * ROWS + t / LPR, tok = pg * KV_PAGE + r;
        if (tok < len || tok >= end) continue;
        *reinterpret_cast<uint4*>(tail_k + r * D + pr.x1) = kx[it];
        *reinterpret_cast<uint4*>(tail_k + r * D + pr.x2) = ky[it];
        const int pl = v_place(r);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          tail_v[(pr.x1 + i) * KV_PAGE + pl] = elem8(vx[it], i);
          tail_v[(pr.x2 + i) * KV_PAGE + pl] = elem8(vy[it], i);
        }
      }
      if (t == 0) {
        // the tokens of an earlier call in this page count too; a NaN stays
        const float old = pg * KV_PAGE < len ? top0 : 0.0f;
        *tail_top = vbad || old != old ? nan : fmaxf(old, vt_);
      }
      return;
    }

    const int pid = a.c.table[(long long)slot * a.c.max_pages + pg];
    if (pid < 0 || pid >= a.c.n_pages) {
      if (t == 0) atomicOr(a.c.status, KV_ST_PAGE);
      return;
    }
    constexpr float M = code_max<CODES>();
    const float kinv = kbad || kt == 0.0f ? 0.0f : fminf(M / kt, 0x1.fffffep127f);
    const float vinv = vbad || vt_ == 0.0f ? 0.0f : fminf(M / vt_, 0x1.fffffep127f);
    const long long at = (long long)pid * H + h;
    uint8_t* kc = reinterpret_cast<uint8_t*>(a.c.k_codes) + at * KV_PAGE * D;
    uint8_t* vc = reinterpret_cast<uint8_t*>(a.c.v_codes) + at * KV_PAGE * D;
    auto codes = [&](const uint4& x, float inv, bool bad) {
      if (bad) return make_uint2(0u, 0u);
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = Elem<DT>::get(elem8(x, i)) * inv;
      return make_uint2(narrow4<CODES>(y[0], y[1], y[2], y[3]), narrow4<CODES>(y[4], y[5], y[6], y[7]));
    };
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int r = it * ROWS + t / LPR;
      *reinterpret_cast<uint2*>(kc + r * D + pr.x1) = codes(kx[it], kinv, kbad);
      *reinterpret_cast<uint2*>(kc + r * D + pr.x2) = codes(ky[it], kinv, kbad);
      const uint2 c1 = codes(vx[it], vinv, vbad), c2 = codes(vy[it], vinv, vbad);
      const int pl = v_place(r);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        vt[(pr.x1 + i) * VROW + pl] = (uint8_t)((i < 4 ? c1.x : c1.y) >> (8 * (i & 3)));
        vt[(pr.x2 + i) * VROW + pl] = (uint8_t)((i < 4 ? c2.x : c2.y) >> (8 * (i & 3)));
      }
    }
    if (t == 0) {
      a.c.k_scale[at] = kbad ? nan : kt * (1.0f / M);
      a.c.v_scale[at] = vbad ? nan : vt_ * (1.0f / M);
      if (kbad || vbad) atomicOr(a.c.status, KV_ST_NONFINITE);
    }
    __syncthreads();
    for (int i = t; i < D * KV_PAGE / 16; i += THREADS) {
      const uint32_t* s = reinterpret_cast<const uint32_t*>(vt + (i >> 2) * VROW + (i & 3) * 16);
      *reinterpret_cast<uint4*>(vc + i * 16) = make_uint4(s[0], s[1], s[2], s[3]);
    }
  };

  if (part == 0 && p1 == p0 && a.n < KV_PAGE) {
    uint32_t top = 0;
    for (int i = mine; i < end - len; i += ROWS) {
      if (i != mine) token(i, kx0, ky0, vx0, vy0);
      const int r = len - p0 * KV_PAGE + i, pl = v_place(r);
      *reinterpret_cast<uint4*>(tail_k + r * D + pr.x1) = kx0;
      *reinterpret_cast<uint4*>(tail_k + r * D + pr.x2) = ky0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        tail_v[(pr.x1 + j) * KV_PAGE + pl] = elem8(vx0, j);
        tail_v[(pr.x2 + j) * KV_PAGE + pl] = elem8(vy0, j);
      }
      top = top_bits(vy0, top_bits(vx0, top));
    }
    top = wave_max_u32(top);
    if ((t & 63) == 0) red[0][t >> 6] = top;
    __syncthreads();
    if (t == 0 && end > len) {
#pragma unroll
      for (int w = 1; w < THREADS / 64; ++w) top = max(top, red[0][w]);
      const float old = p0 * KV_PAGE < len ? top0 : 0.0f;
      *tail_top = top >= Elem<DT>::INF || old != old ? __uint_as_float(0x7fc00000u)
                                                     : fmaxf(old, Elem<DT>::get((uint16_t)top));
    }
  } else if (part == 0) {
    if (p1 > p0) page(p0, true);
    if (end > max(len, p1 * KV_PAGE)) page(p1, false);
  } else if (p0 + part < p1) {
    page(p0 + part, true);
  }

  if (outside) atomicOr(a.c.status, KV_ST_POS);
  // The last workgroup of the sequence to finish moves its length on: each has read it by then.
  __syncthreads();
  if (t == 0) {
    const int all = a.pages * H;
    int* arrived = a.c.arrived + (long long)slot * KV_LINE;  // a line of its own: sharing one cost 6 ns an arrival
    if (atomicAdd(arrived, 1) == all - 1) {
      *arrived = 0;
      a.c.lens[slot] = end;
    }
  }
}

// Tokens start..start+n-1 of each sequence in 16 bits (zeros before its first and past its last).
// One workgroup per page that the window can touch and head: codes transposed through LDS. Bound by memory (8 x 1,000
// tokens of 24 heads of 64: 14 us for 70 MB, 5 TB/s).
template <int DT, int CODES, int D>
__global__ __launch_bounds__(THREADS) void k_kv_read(ress_kv_cache c, const int* __restrict__ slots,
                                                     const int* __restrict__ start, int n, int pages,
                                                     uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out) {
  constexpr int VROW = KV_PAGE + 4;
  __shared__ __align__(16) uint16_t vt[D * VROW];
  const int t = threadIdx.x, H = c.kv_heads;
  const int part = blockIdx.x % pages, h = blockIdx.x / pages % H, b = blockIdx.x / pages / H;
  bool there;
  const int slot = slot_of(c, slots, b, there);
  const int len = held_tokens(c.lens[slot], there ? c.max_pages : 0);
  const long long s0 = start ? start[b] : (long long)len - n;
  const long long first = (s0 >= 0 ? s0 : s0 - (KV_PAGE - 1)) / KV_PAGE * KV_PAGE;  // of the window's first page
  const long long lo = first + (long long)part * KV_PAGE;
  if (lo >= s0 + n) return;
  const int pg = (int)(lo / KV_PAGE);
  const bool any = lo >= 0 && lo < len, open = any && pg == len / KV_PAGE;
  int pid = -1;
  if (any && !open && pg < c.max_pages) {
    pid = c.table[(long long)slot * c.max_pages + pg];
    if (pid < 0 || pid >= c.n_pages) {
      if (t == 0) atomicOr(c.status, KV_ST_PAGE);
      pid = -1;
    }
  }
  const long long at = (long long)pid * H + h;
  const long long tail = ((long long)slot * H + h) * KV_PAGE * D;
  const float ks = pid >= 0 ? c.k_scale[at] : 0.0f, vs = pid >= 0 ? c.v_scale[at] : 0.0f;
  // the keys on their way, then the page's values, rows of 64 places in their order, into LDS
  constexpr int KI = KV_PAGE * D / 8 / THREADS;
  uint2 kc[KI];
#pragma unroll
  for (int j = 0; j < KI; ++j)
    if (pid >= 0)
      kc[j] = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(c.k_codes) + at * KV_PAGE * D + (t + j * THREADS) * 8);
  for (int i = t; i < D * KV_PAGE / 8; i += THREADS) {
    const int d = i >> 3, p = (i & 7) * 8;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (open) {
      w = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(c.tail_v) + tail + d * KV_PAGE + p);
    } else if (pid >= 0) {
      const uint2 cv = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(c.v_codes) + at * KV_PAGE * D + d * KV_PAGE + p);
      uint16_t e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = Elem<DT>::put(code_value<CODES>((uint8_t)((j < 4 ? cv.x : cv.y) >> (8 * (j & 3)))) * vs);
      w = pack8(e);
    }
    uint32_t* dst = reinterpret_cast<uint32_t*>(vt + d * VROW + p);
    dst[0] = w.x; dst[1] = w.y; dst[2] = w.z; dst[3] = w.w;
  }
  __syncthreads();
#pragma unroll
  for (int it = 0; it < KI; ++it) {
    const int i = t + it * THREADS, r = i / (D / 8), d = (i % (D / 8)) * 8;
    const long long tok = lo + r;
    if (tok < s0 || tok >= s0 + n) continue;
    uint4 kw = make_uint4(0, 0, 0, 0), vw = kw;
    if (any && tok < len) {
      if (open) {
        kw = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(c.tail_k) + tail + r * D + d);
      } else if (pid >= 0) {
        const uint2 cv = kc[it];
        uint16_t e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = Elem<DT>::put(code_value<CODES>((uint8_t)((j < 4 ? cv.x : cv.y) >> (8 * (j & 3)))) * ks);
        kw = pack8(e);
      }
      uint16_t e[8];
      const int pl = v_place(r);
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = vt[(d + j) * VROW + pl];
      vw = pack8(e);
    }
    const long long o = (((long long)b * H + h) * n + (tok - s0)) * D + d;
    *reinterpret_cast<uint4*>(k_out + o) = kw;
    *reinterpret_cast<uint4*>(v_out + o) = vw;
  }
  if (!there && t == 0) atomicOr(c.status, KV_ST_SLOT);  // at the end: it would hold up the loads
}

template <template <int, int, int> class Launch, class... A>
int by_kind(const ress_kv_cache& c, A&&... args) {
  const bool f16 = c.dtype == KV_F16, fp8 = c.codes == KV_FP8;
  if (c.head_dim == 64) {
    if (f16) return fp8 ? Launch<KV_F16, KV_FP8, 64>::go(args...) : Launch<KV_F16, KV_I8, 64>::go(args...);
    return fp8 ? Launch<KV_BF16, KV_FP8, 64>::go(args...) : Launch<KV_BF16, KV_I8, 64>::go(args...);
  }
  if (f16) return fp8 ? Launch<KV_F16, KV_FP8, 128>::go(args...) : Launch<KV_F16, KV_I8, 128>::go(args...);
  return fp8 ? Launch<KV_BF16, KV_FP8, 128>::go(args...) : Launch<KV_BF16, KV_I8, 128>::go(args...);
}

template <int DT, int CODES, int D>
struct Append {
  static int go(const AppendArgs& a, hipStream_t stream) {
    const long long kv = (long long)a.B * a.c.kv_heads * a.pages;
    const long long qg = a.q_out ? (long long)a.B * cdiv(a.Hq, QH) * cdiv(a.n, THREADS / (D / 16)) : 0;
    RESS_REQUIRE(launchable(kv + qg, THREADS), "ress_kv_append: the call needs 2^32 threads or more");
    hipLaunchKernelGGL((k_kv_append<DT, CODES, D>), dim3((unsigned)(kv + qg)), dim3(THREADS), 0, stream, a, (int)kv);
    RESS_LAUNCHED("k_kv_append");
    return 0;
  }
};

template <int DT, int CODES, int D>
struct Read {
  static int go(const ress_kv_cache& c, int B, int n, const int* slots, const int* start, void* k, void* v,
                hipStream_t stream) {
    const int pages = (n + KV_PAGE - 1) / KV_PAGE + 1;
    const long long g = (long long)B * c.kv_heads * pages;
    RESS_REQUIRE(launchable(g, THREADS), "ress_kv_read: the call needs 2^32 threads or more");
    hipLaunchKernelGGL((k_kv_read<DT, CODES, D>), dim3((unsigned)g), dim3(THREADS), 0, stream, c, slots, start, n,
                       pages, (uint16_t*)k, (uint16_t*)v);
    RESS_LAUNCHED("k_kv_read");
    return 0;
  }
};

bool multiple(long long a, long long b, long long c, int m) { return a % m == 0 && b % m == 0 && c % m == 0; }

}  // namespace

int ress_kv_check(const ress_kv_cache* c, int B, const char* who) {
  RESS_REQUIRE(c, "%s: null cache", who);
  RESS_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "%s: head_dim %d is not 64 or 128", who, c->head_dim);
  RESS_REQUIRE(c->dtype == KV_BF16 || c->dtype == KV_F16, "%s: dtype code %d is not 1 (bf16) or 2 (fp16)", who, c->dtype);
  RESS_REQUIRE(c->codes == KV_I8 || c->codes == KV_FP8, "%s: codes %d is not 0 (int8) or 1 (e4m3)", who, c->codes);
  RESS_REQUIRE(c->n_pages > 0 && c->max_pages > 0 && c->max_seqs > 0 && c->kv_heads > 0 &&
                   c->max_pages < (1 << 25),  // tokens are counted in 32 bits
               "%s: bad cache geometry", who);
  RESS_REQUIRE(c->k_codes && c->v_codes && c->k_scale && c->v_scale && c->tail_k && c->tail_v && c->tail_top &&
                   c->table && c->held && c->lens && c->arrived && c->status,
               "%s: the cache has a null buffer", who);
  RESS_REQUIRE(((uintptr_t)c->k_codes | (uintptr_t)c->v_codes | (uintptr_t)c->tail_k | (uintptr_t)c->tail_v) % 16 == 0,
               "%s: the cache's buffers are not 16-byte aligned", who);
  RESS_REQUIRE(B >= 0 && B <= c->max_seqs, "%s: batch %d is more than the cache's %d slots", who, B, c->max_seqs);
  return 0;
}

RESS_API int ress_kv_append(const ress_kv_cache* cache, const void* k, long long skB, long long skH, long long skT,
                            const void* v, long long svB, long long svH, long long svT, const void* q, long long sqB,
                            long long sqH, long long sqT, int B, int Hq, int n, const long long* pos,
                            const float* rope, int positions, int axes, const int* slots, const int* new_lens,
                            void* q_out, hipStream_t stream) {
  if (int rc = ress_kv_check(cache, B, "ress_kv_append")) return rc;
  RESS_REQUIRE(n >= 0 && n <= (1 << 30) && Hq >= 0, "ress_kv_append: bad sizes (n %d, query heads %d)", n, Hq);
  RESS_REQUIRE(!q == !q_out, "ress_kv_append: q and q_out go together");
  RESS_REQUIRE(!q || pos, "ress_kv_append: queries without positions");
  RESS_REQUIRE(!pos || (rope && positions > 0 && (axes == 1 || axes == 2)),
               "ress_kv_append: positions need a table of at least one row and 1 or 2 axes");
  if (B == 0 || n == 0) return 0;
  RESS_REQUIRE(k && v, "ress_kv_append: null keys or values");
  AppendArgs a{};
  a.c = *cache;
  a.k = (const uint16_t*)k; a.v = (const uint16_t*)v; a.q = (const uint16_t*)q;
  a.skb = skB; a.skh = skH; a.skt = skT; a.svb = svB; a.svh = svH; a.svt = svT; a.sqb = sqB; a.sqh = sqH; a.sqt = sqT;
  a.pos = pos; a.rope = rope; a.positions = positions; a.axes = pos ? axes : 1;
  a.B = B; a.Hq = q ? Hq : 0; a.n = n; a.slots = slots; a.new_lens = new_lens; a.q_out = (uint16_t*)q_out;
  a.pages = (n + KV_PAGE - 1) / KV_PAGE;  // pages filled, at most (one more, the last, goes with the first)
  a.vec = ((uintptr_t)k | (uintptr_t)v | (uintptr_t)q) % 16 == 0 && multiple(skB, skH, skT, 8) &&
          multiple(svB, svH, svT, 8) && (!q || multiple(sqB, sqH, sqT, 8));
  return by_kind<Append>(a.c, a, stream);
}

RESS_API int ress_kv_read(const ress_kv_cache* cache, int B, int n, const int* slots, const int* start, void* k,
                          void* v, hipStream_t stream) {
  if (int rc = ress_kv_check(cache, B, "ress_kv_read")) return rc;
  RESS_REQUIRE(n >= 0 && n <= (1 << 30), "ress_kv_read: bad token count %d", n);
  if (B == 0 || n == 0) return 0;
  RESS_REQUIRE(k && v && ((uintptr_t)k | (uintptr_t)v) % 16 == 0, "ress_kv_read: outputs null or not 16-byte aligned");
  return by_kind<Read>(*cache, *cache, B, n, slots, start, k, v, stream);
}
