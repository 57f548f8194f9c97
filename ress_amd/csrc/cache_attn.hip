// Attention over the paged 8-bit key/value cache (layout: kvcache.h).
//
// o = softmax(s q K^T) V with K = code * k_scale, V = code * v_scale per (page, head). With 16x16x32
// MFMAs and the operands transposed, S^T = K Q^T (A = codes of 16 keys, B = 16 queries) and
// O^T += V^T P^T (A = values of 16 dims), a lane holds for ITS query four keys of each 16, which is what
// the second product takes as its B operand once the keys of a value row are stored in that order (v_token): P
// never leaves the registers. The codes are widened to 16 bits exactly; the scales of a page multiply
// the scores (folded into the exponent's multiply-add) and P or the values (below). Rounded to 16 bits are P, in fp16 each
// value (code * v_scale) too, and the output. Max, sum and output accumulate in fp32.
//
// Running max. m starts at the lowest finite value and moves only when a score of the wave lies more than
// LAZY = 8 (in log2) above its row's m: P is then at most 2^8, sums are unaffected, and most pages need
// neither the exchange between a row's four lanes nor a pass over the accumulators.
//
// v_scale. In bf16 it enters as an addend of the exponent (PageScale), relative to a power of two: the codes stay whole
// and it costs no multiplication per element. fp16 has no exponents to spare for that: there the codes are multiplied,
// as they are widened, by v_scale rounded toward zero to fp16 (the products are rounded to fp16, in whose range they are as the
// values they came from were; a scale below 2^-14, which fp16 holds with fewer bits, goes to the nearest), and what the
// scale's rounding took or added enters the exponent.
// The sum of P is a product with ones on the matrix cores, of the rounded P, so numerator and denominator carry the
// same roundings.
//
// Masked places (past the sequence's end, after the row's own token) are selected away after every
// multiplication, so a NaN scale or tail element there reaches no row that does not see its page.
#include "kvcache.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr float LOWEST = -0x1.fffffep127f;
constexpr int CUS = 256;
constexpr float LAZY = 8.0f;

struct AttendArgs {
  ress_kv_cache c;
  const uint16_t* q;
  uint16_t* out;
  long long sqb, sqh, sqt, sob, soh, sot;
  int B, Hq, n, G;   // G = Hq / kv_heads
  const int *slots, *new_lens;
  int causal;
  float scale;       // sm_scale * log2(e)
  int splits, per;   // the keys are cut every `per` pages, into at most `splits` parts (the last takes the rest)
  int tiles;         // row tiles of a (sequence, kv head)
  float *part_o, *part_ml;  // [splits][B * kv_heads * n * G][D] outputs of the parts, [..][2] their m and l
  bool qvec, ovec;
};

template <int DT>
__device__ __forceinline__ v4f mfma(const uint4& a, const uint4& b, const v4f& c) {
  if constexpr (DT == KV_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (DT == KV_BF16) {
    const v2bf r = {(__bf16)lo, (__bf16)hi};
    return __builtin_bit_cast(uint32_t, r);
  } else {
    const v2h r = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, r);
  }
}

// The arrays that are only read, as parameters of their own: the compiler then takes page numbers and scales by
// scalar loads (a member of the argument struct might be written through another, and goes through vector registers).
#define RESS_READ_ONLY                                                                                           \
  const int *__restrict__ table_all, const float *__restrict__ k_scale, const float *__restrict__ v_scale, \
      const int *__restrict__ lens, const int *__restrict__ slots, const int *__restrict__ new_lens

// One sequence and key/value head: what it holds.
template <int D>
struct Head {
  int len, nv, slot, h;
  bool there;                  // the slot lies in the cache
  const uint8_t *kc, *vc;      // codes of page 0 of this head
  const uint16_t *tk, *tv;     // the unfinished page
  long long stride;            // bytes from page to page
  __device__ __forceinline__ Head(const AttendArgs& a, const int* __restrict__ lens, const int* __restrict__ slots,
                                  const int* __restrict__ new_lens, int b, int h_) : h(h_) {
    slot = slot_of(a.c, slots, b, there);
    len = there ? held_tokens(lens[slot], a.c.max_pages) : 0;  // bounded by 0 pages instead, 512 causal rows at a head of 128 took 150 us for 145
    nv = new_lens ? min(max(new_lens[b], 0), a.n) : a.n;
    const long long one = (long long)KV_PAGE * D;
    kc = reinterpret_cast<const uint8_t*>(a.c.k_codes) + h * one;
    vc = reinterpret_cast<const uint8_t*>(a.c.v_codes) + h * one;
    tk = reinterpret_cast<const uint16_t*>(a.c.tail_k) + ((long long)slot * a.c.kv_heads + h) * one;
    tv = reinterpret_cast<const uint16_t*>(a.c.tail_v) + ((long long)slot * a.c.kv_heads + h) * one;
    stride = one * a.c.kv_heads;
  }
};

// The unfinished page's values as the second product takes them. bf16: scaled by a power of two to at most 128 (like
// codes), undone by its v_scale, so that it does not set R off. fp16: as they are. NaN v_scale (and values 0) where one
// is not finite.
template <int DT>
struct TailScale {
  float down, vs;  // multiply the values by down, P by vs
  __device__ __forceinline__ explicit TailScale(float top) {
    const bool bad = top != top;
    int e = 0;
    if (DT == KV_BF16 && !bad && top > 0.0f) {
      frexpf(top, &e);  // top < 2^e
      e = min(max(e - 7, -100), 100);
    }
    down = bad ? 0.0f : ldexpf(1.0f, -e);
    vs = bad ? __uint_as_float(0x7fc00000u) : ldexpf(1.0f, e);
  }
};

// How a page's v_scale enters P: P comes out of the exponential times 2^lift, and its sum is multiplied by `down` again.
// bf16: relative to R = 2^eR, a power of two at least as large as any v_scale met so far (exact to rescale by, so a row's
// bits do not hang on the pages that only its neighbours see); at most 2^-60 of R is lost to the clamp (a page of
// zeros has v_scale 0). fp16: P is lifted by 2^7 (it is at most 2^LAZY, so below 2^15), which the quotient of the sums
// takes out again, and carries v_scale / value_scale(v_scale).
template <int DT>
__device__ __forceinline__ float value_scale(float vs) {
  if constexpr (DT == KV_BF16) return 1.0f;
  // toward zero, as 127 times the nearest of 65504 / 127 is infinite (what the mask leaves of a subnormal the cast rounds to
  // nearest); never 0 (the smallest subnormal serves the smallest scales), so that 0 * V is 0
  return vs > 0.0f ? fmaxf((float)(_Float16)__uint_as_float(__float_as_uint(vs) & 0xffffe000u), 0x1p-24f) : 1.0f;
}
template <int DT>
struct PageScale {
  float lift, down;
  __device__ __forceinline__ PageScale(float vs, int eR) {
    if constexpr (DT == KV_F16) {
      const float r = vs == 0.0f ? 1.0f : vs / value_scale<DT>(vs);  // below 1 + 2^-10, of subnormals below 2; NaN stays
      lift = 7.0f + __builtin_amdgcn_logf(r);
      down = 1.0f / r;
    } else {
      const float q = __builtin_amdgcn_logf(ldexpf(vs, -eR));  // log2
      lift = q < -60.0f ? -60.0f : q;                          // NaN stays
      down = __builtin_amdgcn_exp2f(-lift);
    }
  }
};

// A lane's state for CT tiles of 16 queries: query 16 ct + (lane & 15), shared by the four lanes of a column.
template <int DT, int D, int CT>
struct Rows {
  v4f o[CT][D / 16];   // dims 16 dt + 4 (lane >> 4) + r; bf16: relative to 2^eR
  float m[CT], l[CT];
  int eR;
  __device__ __forceinline__ void clear() {
    eR = -120;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      m[c] = LOWEST;
      l[c] = 0.0f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[c][d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }

  // Scores s of 64 keys -> P as the second product's B operand p. cs = k_scale * sm_scale * log2(e). MASK: query c sees the tile's keys below lim[c].
  template <bool MASK>
  __device__ __forceinline__ void softmax(const v4f (&s)[CT][4], float cs, float vs, const int (&lim)[CT], int h4,
                                          uint4 (&p)[CT][2]) {
    int below[CT];  // the lane's keys 16 k + 4 h4 + r that are seen: 16 k + r < below
#pragma unroll
    for (int c = 0; c < CT; ++c) below[c] = lim[c] - 4 * h4;
    auto highest = [&](int c) {  // of the lane's scores of row c, times cs
      float t = LOWEST;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x = s[c][k][r];
          if constexpr (MASK) x = 16 * k + r < below[c] ? x : -__builtin_huge_valf();
          t = fmaxf(t, x);
        }
      return MASK && t == LOWEST ? LOWEST : t * cs;
    };
    // Whether a score lies more than LAZY above its row's m. Where m + LAZY is not negative only positive scores can,
    // and they order as their bits do: integer maxima, which need no pass that quiets NaNs.
    bool up = false, below0 = false;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      int t = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          int x = __float_as_int(s[c][k][r]);
          if constexpr (MASK) x = 16 * k + r < below[c] ? x : 0;
          t = max(t, x);
        }
      up = up || __int_as_float(t) * cs > m[c] + LAZY;
      below0 = below0 || m[c] + LAZY < 0.0f;
    }
    if (__any(up || below0)) {
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        float t = fmaxf(highest(c), m[c]);
        t = fmaxf(t, xor_lane_f<16>(t));
        t = fmaxf(t, xor_lane_f<32>(t));
        t = t > m[c] + LAZY ? t : m[c];  // a row moves by its own scores, so its bits do not hang on its neighbours
        const float a = exp2f(m[c] - t);
        m[c] = t;
        l[c] *= a;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) o[c][d] *= a;
      }
    }
    if (DT == KV_BF16 && vs > ldexpf(1.0f, eR)) {
      const int e = (int)((__float_as_uint(vs) + 0x7fffffu) >> 23) - 127;  // vs <= 2^e
      const float a = ldexpf(1.0f, eR - e);
      eR = e;
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int d = 0; d < D / 16; ++d) o[c][d] *= a;
    }
    const PageScale<DT> ps(vs, eR);
    const uint4 ones = DT == KV_F16 ? make_uint4(0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u)
                                    : make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      uint32_t w[8];
      const float off = ps.lift - m[c];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float e[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          e[r] = __builtin_amdgcn_exp2f(fmaf(s[c][k][r], cs, off));
          if constexpr (MASK) e[r] = 16 * k + r < below[c] ? e[r] : 0.0f;
        }
        w[2 * k] = pack2<DT>(e[0], e[1]);
        w[2 * k + 1] = pack2<DT>(e[2], e[3]);
      }
      p[c][0] = make_uint4(w[0], w[1], w[2], w[3]);
      p[c][1] = make_uint4(w[4], w[5], w[6], w[7]);
      // the row's sum over the page, in every lane of its column: a product with ones
      v4f t = {0.0f, 0.0f, 0.0f, 0.0f};
      t = mfma<DT>(ones, p[c][0], t);
      t = mfma<DT>(ones, p[c][1], t);
      l[c] = MASK && lim[c] <= 0 ? l[c] : fmaf(t[0], ps.down, l[c]);  // 0 * NaN would not be 0
    }
  }

  // o of dims 16 d.. += P V, the page's values as the A operands a (32 keys each)
  __device__ __forceinline__ void add(int d, const uint4& a0, const uint4& a1, const uint4 (&p)[CT][2]) {
#pragma unroll
    for (int c = 0; c < CT; ++c) o[c][d] = mfma<DT>(a1, p[c][1], mfma<DT>(a0, p[c][0], o[c][d]));
  }

  // The factor that takes o to its own units
  __device__ __forceinline__ float unit() const { return DT == KV_F16 ? 1.0f : ldexpf(1.0f, eR); }
};

// Row r of a (sequence, kv head): token r / G, query head h G + r % G.
template <int D, int CT>
__device__ __forceinline__ void load_q(const AttendArgs& a, int b, int h, int row0, int rows, int lane,
                                       uint4 (&qv)[CT][D / 32]) {
  const int h4 = lane >> 4;
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int r = row0 + 16 * c + (lane & 15);
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      qv[c][s] = make_uint4(0, 0, 0, 0);
      if (r < rows) {  // dims of step s: 64 (s / 2) + 16 h4 + 8 (s % 2) + 0..7, as the codes are read
        const int tok = r / a.G, hq = h * a.G + r % a.G;
        qv[c][s] = ld8(a.q + b * a.sqb + hq * a.sqh + tok * a.sqt + 64 * (s >> 1) + 16 * h4 + 8 * (s & 1), a.qvec);
      }
    }
  }
}

// Twice `half`, a weighted mean of values over two. No mean passes the type's largest value, but the weights and v_scale are
// rounded by 2^-9 (bf16) or 2^-11, so its sum may: it ends there. Infinities and NaN stay.
template <int DT>
__device__ __forceinline__ v4f mean4(const v4f& half) {
  constexpr float TOP = DT == KV_F16 ? 0.5f * 65504.0f : 0x0.ffp127f;
  v4f r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = fabsf(half[i]);
    r[i] = 2.0f * (x > TOP && x < __builtin_inff() ? copysignf(TOP, half[i]) : half[i]);
  }
  return r;
}

template <int DT>
__device__ __forceinline__ void store4(uint16_t* p, const v4f& v, bool vec) {
  const uint32_t lo = pack2<DT>(v[0], v[1]), hi = pack2<DT>(v[2], v[3]);
  if (vec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(lo, hi);
  } else {
    p[0] = (uint16_t)lo; p[1] = (uint16_t)(lo >> 16); p[2] = (uint16_t)hi; p[3] = (uint16_t)(hi >> 16);
  }
}

// 16 codes (two steps' operands) widened
template <int DT, int CODES>
__device__ __forceinline__ void widen16(const uint4& w, uint4& a, uint4& b) {
  const uint2 x = widen4<DT, CODES>(w.x), y = widen4<DT, CODES>(w.y), z = widen4<DT, CODES>(w.z), u = widen4<DT, CODES>(w.w);
  a = make_uint4(x.x, x.y, y.x, y.y);
  b = make_uint4(z.x, z.y, u.x, u.y);
}
// 16 codes of values widened, times value_scale (fp16: one more packed multiplication for two)
template <int DT, int CODES>
__device__ __forceinline__ void widen16_v(const uint4& w, float scale, uint4& a, uint4& b) {
  widen16<DT, CODES>(w, a, b);
  if constexpr (DT == KV_F16) {
    const v2h m = {(_Float16)scale, (_Float16)scale};
    auto times = [&](uint32_t& x) { x = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, x) * m); };
    times(a.x); times(a.y); times(a.z); times(a.w);
    times(b.x); times(b.y); times(b.z); times(b.w);
  }
}
// A lane's values of the unfinished page: its 16 places (16 h4 on) of a dim, two a word. keep[] clears those of tokens from
// cnt on (all of them with down = 0); bf16: times the power of two `down` (exact but for values 2^-126 and less, which are
// cut off). Two words' worth of instructions a word: this code runs once a call, mostly as fast as it is fetched (with
// conversions and comparisons an element, and loads as they were needed, a call took 4 to 14 us more: 4 sequences of 1,000
// tokens, 32 heads over 8 of 128, 25 us instead of 13).
template <int DT>
struct TailValues {
  uint32_t keep[8];
  float down;
  __device__ __forceinline__ TailValues(float down_, int h4, int cnt) : down(down_) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = v_token(2 * i) + 4 * h4;  // v_token(16 h4 + 2 i); the next place is the next token
      keep[i] = down == 0.0f ? 0u : t + 1 < cnt ? ~0u : t < cnt ? 0xffffu : 0u;
    }
  }
  __device__ __forceinline__ uint32_t pair(uint32_t w, int i) const {
    w &= keep[i];
    if constexpr (DT == KV_F16) return w;
    const float lo = __uint_as_float(w << 16) * down, hi = __uint_as_float(w & 0xffff0000u) * down;
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
  }
  __device__ __forceinline__ uint4 half(const uint4& w, int i) const {  // places 8 i on
    return make_uint4(pair(w.x, 4 * i), pair(w.y, 4 * i + 1), pair(w.z, 4 * i + 2), pair(w.w, 4 * i + 3));
  }
};

// Waves that a SIMD's registers are shared out for. One more spills: us a call for one row of 16 heads of 64 over 21,984
// tokens 17.3 instead of 17.1, five over 274,800 109 instead of 102, 32 sequences of up to 8,192 tokens, 8 heads of 128, 153
// instead of 63; with 32 rows and a head of 128 two spill.
constexpr int few_waves(int D, int CT) { return CT == 2 ? (D == 64 ? 2 : 1) : D == 64 ? 3 : 2; }

// ---- few rows: one wave a page --------------------------------------------------------------------
// A workgroup of four waves takes 16 CT rows of a (sequence, kv head) and a share of its pages, a wave every
// fourth page, codes straight from memory into the operands (1 KB, contiguous, an access). The waves' parts are
// joined in LDS. Bound by the bytes of the codes where the cache is long (5 rows of 16 heads over 274,800 tokens: 96 us
// for 563 MB, 5.9 TB/s), by one page's chain of loads, scores, exponentials and products where it is short (one row over
// 21,984 tokens: 12 us, 3.8 TB/s; the call takes 16, its parts being joined in 4).
template <int DT, int CODES, int D, int CT>
__global__ __launch_bounds__(256, few_waves(D, CT)) void k_cache_attn_few(AttendArgs a, RESS_READ_ONLY) {
  constexpr int NW = 4;
  constexpr int TILES = CT * D / 16;  // of the output: 16 queries, 16 dims
  __shared__ v4f so[NW][TILES][64];
  __shared__ float sm[NW][CT][16], sl[NW][CT][16];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h4 = lane >> 4;
  // heads vary fastest, so every XCD gets as much of each part (the last is shorter, and short sequences have fewer)
  const int H = a.c.kv_heads, bh = blockIdx.x % (a.B * H), split = blockIdx.x / (a.B * H) % a.splits;
  const int tile = blockIdx.x / (a.B * H) / a.splits, b = bh / H, h = bh % H;
  const Head<D> hd(a, lens, slots, new_lens, b, h);
  const int rows = hd.nv * a.G, row0 = tile * 16 * CT;
  const long long all_rows = (long long)a.B * H * a.n * a.G;
  if (row0 >= rows) return;
  uint4 qv[CT][D / 32];
  load_q<D, CT>(a, b, h, row0, rows, lane, qv);

  const int* __restrict__ table = table_all + (long long)hd.slot * a.c.max_pages;
  constexpr int KU = D / 16, VU = D / 16;  // 1 KB units of a page: keys (4 tiles x D / 64 halves), values (D / 16)
  // A page's codes are loaded as soon as the registers are free: the next one's keys behind the scores, its values
  // behind P V; its number a page ahead of them. The first page's are on their way before the length is known (they are
  // not used where it has none). A bad page number reads as a page of zeros.
  uint4 kw[KU], vw[VU];
  float ks = 0.0f, vs = 0.0f;
  int bad = 0;
  auto number = [&](int pg) { return pg < a.c.max_pages ? table[pg] : -1; };
  auto there = [&](int id) { return id >= 0 && id < a.c.n_pages; };
  const unsigned k0 = (lane & 15) * (D / 16) + h4, v0 = (lane & 15) * 4 + h4;  // in 16-byte pieces
  auto load_k = [&](int id) {
    const int pid = there(id) ? id : 0;
    const uint4* p = reinterpret_cast<const uint4*>(hd.kc + pid * hd.stride);
#pragma unroll
    for (int u = 0; u < KU; ++u) kw[u] = at_u32(p, k0 + u / (D / 64) * D + u % (D / 64) * 4);
    ks = there(id) ? k_scale[(long long)pid * H + h] : 0.0f;
  };
  auto load_v = [&](int id) {
    const int pid = there(id) ? id : 0;
    const uint4* p = reinterpret_cast<const uint4*>(hd.vc + pid * hd.stride);
#pragma unroll
    for (int u = 0; u < VU; ++u) vw[u] = at_u32(p, v0 + u * 64);
    vs = there(id) ? v_scale[(long long)pid * H + h] : 0.0f;
  };
  int id = number(split * a.per + w), next = number(split * a.per + w + NW);
  load_k(id);
  load_v(id);

  const int full = hd.len / KV_PAGE, left = hd.len % KV_PAGE, pages = full + (left ? 1 : 0);
  const int parts = min(a.splits, cdiv(pages, a.per));
  const int lo = min(pages, split * a.per), hi = split == a.splits - 1 ? pages : min(pages, lo + a.per);
  if (split && lo >= pages) return;  // the join goes by the same count
  int limit[CT];  // tokens that the lane's query sees
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int tok = (row0 + 16 * c + (lane & 15)) / a.G;
    limit[c] = a.causal ? max(0, hd.len - hd.nv + tok + 1) : hd.len;
  }
  const int seen_by_all = a.causal ? max(0, hd.len - hd.nv + row0 / a.G + 1) : hd.len;
  const int seen_by_any =
      a.causal ? max(0, hd.len - hd.nv + (min(row0 + 16 * CT, rows) - 1) / a.G + 1) : hd.len;

  Rows<DT, D, CT> st;
  st.clear();
  auto weights = [&](const v4f (&s)[CT][4], float cs, float v, int pg, uint4 (&p)[CT][2]) {
    int lim[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) lim[c] = limit[c] - pg * KV_PAGE;
    if (pg * KV_PAGE + KV_PAGE <= seen_by_all) st.template softmax<false>(s, cs, v, lim, h4, p);
    else st.template softmax<true>(s, cs, v, lim, h4, p);
  };

  const int last = min(min(hi, full), cdiv(seen_by_any, KV_PAGE));
  for (int pg = lo + w; pg < last; pg += NW) {
    bad |= !there(id);
    const int after = pg + 2 * NW < last ? number(pg + 2 * NW) : -1;
    v4f s[CT][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int c = 0; c < CT; ++c) s[c][k] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < D / 64; ++e) {
        uint4 x, y;
        widen16<DT, CODES>(kw[k * (D / 64) + e], x, y);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          s[c][k] = mfma<DT>(x, qv[c][2 * e], s[c][k]);
          s[c][k] = mfma<DT>(y, qv[c][2 * e + 1], s[c][k]);
        }
      }
    }
    const float cs = ks * a.scale, v = vs;
    if (pg + NW < last) load_k(next);
    uint4 p[CT][2];
    weights(s, cs, v, pg, p);
    const float vscale = value_scale<DT>(v);
#pragma unroll
    for (int d = 0; d < VU; ++d) {
      uint4 x, y;
      widen16_v<DT, CODES>(vw[d], vscale, x, y);
      st.add(d, x, y, p);
    }
    if (pg + NW < last) load_v(next);
    id = next;
    next = after;
  }
  if (bad && lane == 0) atomicOr(a.c.status, KV_ST_PAGE);
  if (!hd.there && threadIdx.x == 0) atomicOr(a.c.status, KV_ST_SLOT);
  // the unfinished page, by the wave whose turn it would be
  if (left && full >= lo && full < hi && (full - lo) % NW == w && full * KV_PAGE < seen_by_any) {
    // its loads together
    const float top = a.c.tail_top[(long long)hd.slot * H + h];
    uint4 kt[4][D / 32], vt[VU][2];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < D / 32; ++e)
        kt[k][e] = *reinterpret_cast<const uint4*>(hd.tk + (16 * k + (lane & 15)) * D + 64 * (e >> 1) + 16 * h4 + 8 * (e & 1));
#pragma unroll
    for (int d = 0; d < VU; ++d) {
      const uint4* row = reinterpret_cast<const uint4*>(hd.tv + (16 * d + (lane & 15)) * KV_PAGE + 16 * h4);
      vt[d][0] = row[0];
      vt[d][1] = row[1];
    }
    __builtin_amdgcn_sched_barrier(0);
    const TailScale<DT> ts(top);
    const TailValues<DT> tv(ts.down, h4, left);
    v4f s[CT][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int c = 0; c < CT; ++c) s[c][k] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < D / 32; ++e)
#pragma unroll
        for (int c = 0; c < CT; ++c) s[c][k] = mfma<DT>(kt[k][e], qv[c][e], s[c][k]);
    }
    uint4 p[CT][2];
    weights(s, a.scale, ts.vs, full, p);
#pragma unroll
    for (int d = 0; d < VU; ++d) st.add(d, tv.half(vt[d][0], 0), tv.half(vt[d][1], 1), p);
  }

  // join the four waves
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    if (lane < 16) {
      sm[w][c][lane] = st.m[c];
      sl[w][c][lane] = st.l[c];
    }
  }
  __syncthreads();
  float f[CT], M[CT], L[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int i = lane & 15;
    M[c] = fmaxf(fmaxf(sm[0][c][i], sm[1][c][i]), fmaxf(sm[2][c][i], sm[3][c][i]));
    L[c] = 0.0f;
#pragma unroll
    for (int k = 0; k < NW; ++k) L[c] += sl[k][c][i] * exp2f(sm[k][c][i] - M[c]);
    f[c] = L[c] == 0.0f ? 0.0f : exp2f(st.m[c] - M[c]) * (0.5f * st.unit() / L[c]);
  }
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int d = 0; d < D / 16; ++d) so[w][c * (D / 16) + d][lane] = st.o[c][d] * f[c];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < TILES / NW; ++i) {  // wave w's tiles
    const int tile = i * NW + w, c = i * NW / (D / 16), d = tile % (D / 16);
    v4f t = so[0][tile][lane];
#pragma unroll
    for (int k = 1; k < NW; ++k) t += so[k][tile][lane];
    t = mean4<DT>(t);
    const int r = row0 + 16 * c + (lane & 15);
    if (r >= rows) continue;
    const int dim = 16 * d + 4 * h4;
    if (parts <= 1) {
      const int tok = r / a.G, hq = h * a.G + r % a.G;
      store4<DT>(a.out + b * a.sob + hq * a.soh + tok * a.sot + dim, t, a.ovec);
    } else {
      const long long at = split * all_rows + (long long)bh * a.n * a.G + r;
      *reinterpret_cast<v4f*>(a.part_o + at * D + dim) = t;
      if (d == 0 && lane < 16) {
        a.part_ml[2 * at] = M[c];
        a.part_ml[2 * at + 1] = L[c];
      }
    }
  }
}

// ---- many rows: pages widened once for a workgroup ---------------------------------------------------
// NW waves of 16 CT rows each share a page, widened into LDS in the order in which the operands are read (1 KB
// a wave's read, no bank conflicts), the next page's codes loaded meanwhile; two stages, one barrier a page. Pages that
// every row sees whole run without a mask, apart from those that a causal row ends in, so that the masks' registers
// are not held in the loop.
//
// Bound by the vector instructions beside the products: the vector unit is busy 67% of a SIMD's cycles, the matrix cores
// 37% (1,374 rows of 16 heads over 87,936 tokens; a page of 32 rows takes 36 products of 16 cycles, 32 exponentials of 8
// and some 150 other instructions of 4). It issues 0.39 vector instructions a busy matrix cycle where the block-sparse kernel
// (attn.hip), whose products are 32 x 32 and whose exponentials mostly need no maximum, issues 0.15 and keeps the matrix cores
// busy 62%, the vector unit 52%. 495 GFLOP in 630 to 665 us there (cards differ): 740 to 780 TFLOP/s, 36 to 38% of the 2,058
// that the matrix cores reach. Calls at that size and at 21,984 tokens, when they were chosen: 2 tiles of 16 rows a wave 703, 189 us (3: 733,
// 198; 4: 693, 187; 1: 777, 217), four waves a SIMD instead of three 619, 179. Waves of a workgroup: cut().
constexpr int ROWS_CT = 2;
constexpr int rows_waves(int D) { return D == 64 ? 4 : 2; }  // a SIMD; 64 KB of LDS a workgroup at a head of 128

template <int DT, int CODES, int D, int CT, int NW>
__global__ __launch_bounds__(64 * NW, rows_waves(D)) void k_cache_attn_rows(AttendArgs a, RESS_READ_ONLY) {
  constexpr int KU = D / 16, UNITS = 2 * KU;  // 1 KB units of a page's codes: keys, then values
  constexpr int UPW = UNITS / NW;             // of each wave
  static_assert(UPW >= 1 && UPW * NW == UNITS, "every wave has whole units");
  __shared__ uint4 lds[2][UNITS * 128];       // a unit widened: two operand blocks of 1 KB
  const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, h4 = lane >> 4;
  const int H = a.c.kv_heads, groups = a.B * H * a.splits;
  // Workgroups that read the same pages go to one XCD (workgroup i runs on XCD i % 8), and heads vary fastest over the
  // XCDs, as above: 1,374 rows of 16 heads over 21,984 tokens 171 us with the parts' join instead of 177, over 2 sequences of
  // 8,000 and 2,000 tokens 102 instead of 138.
  const int x = blockIdx.x >> 3, group = x / a.tiles * 8 + (blockIdx.x & 7), tile = a.tiles - 1 - x % a.tiles;
  if (group >= groups) return;
  const int split = group / (a.B * H), bh = group % (a.B * H), b = bh / H, h = bh % H;
  const Head<D> hd(a, lens, slots, new_lens, b, h);
  const int rows = hd.nv * a.G, row0 = tile * 16 * CT * NW;
  const long long all_rows = (long long)a.B * H * a.n * a.G;
  if (row0 >= rows) return;
  const int wrow = row0 + 16 * CT * w;
  uint4 qv[CT][D / 32];
  load_q<D, CT>(a, b, h, wrow, rows, lane, qv);

  const int full = hd.len / KV_PAGE, left = hd.len % KV_PAGE, pages = full + (left ? 1 : 0);
  const int before = hd.len - hd.nv;  // causal: row of token i sees before + i + 1 tokens
  auto sees = [&](int r) { return a.causal ? max(0, before + r / a.G + 1) : hd.len; };
  const int parts = min(a.splits, cdiv(pages, a.per));
  const int lo = min(pages, split * a.per);
  if (split && lo >= pages) return;  // the join goes by the same count
  const int hi = min(split == a.splits - 1 ? pages : min(pages, lo + a.per), cdiv(sees(min(row0 + 16 * CT * NW, rows) - 1), KV_PAGE));
  int limit[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) limit[c] = sees(wrow + 16 * c + (lane & 15));
  const int seen_by_any = wrow < rows ? sees(min(wrow + 16 * CT, rows) - 1) : 0;

  Rows<DT, D, CT> st;
  st.clear();
  const int* __restrict__ table = table_all + (long long)hd.slot * a.c.max_pages;
  // Unit u: 16 rows with four 16-code pieces each, lane l taking the piece whose two operands lie at place l of the
  // unit's blocks. Rows of the keys are tokens (D / 16 pieces), of the values dims (4 pieces).
  unsigned piece[UPW];
#pragma unroll
  for (int i = 0; i < UPW; ++i) {
    const int u = w * UPW + i;
    piece[i] = u < KU ? (unsigned)((u / (D / 64) * 16 + (lane & 15)) * (D / 16) + u % (D / 64) * 4 + h4)
                      : (unsigned)(((u - KU) * 16 + (lane & 15)) * 4 + h4);
  }
  uint4 cw[UPW];
  float ks = 0.0f, vs = 0.0f, ks1, vs1;
  int bad = 0;
  auto load = [&](int pg) {
    int pid = pg < a.c.max_pages ? table[pg] : -1;
    const bool ok = pid >= 0 && pid < a.c.n_pages;
    bad |= !ok;
    pid = ok ? pid : 0;
    const uint8_t *kp = hd.kc + pid * hd.stride, *vp = hd.vc + pid * hd.stride;
#pragma unroll
    for (int i = 0; i < UPW; ++i)
      cw[i] = at_u32(reinterpret_cast<const uint4*>(w * UPW + i < KU ? kp : vp), piece[i]);
    const long long at = (long long)pid * H + h;
    ks1 = ok ? k_scale[at] : 0.0f;
    vs1 = ok ? v_scale[at] : 0.0f;
  };
  auto stage = [&](int buf) {
    const float vscale = value_scale<DT>(vs1);
#pragma unroll
    for (int i = 0; i < UPW; ++i) {
      uint4 x, y;
      widen16_v<DT, CODES>(cw[i], w * UPW + i < KU ? 1.0f : vscale, x, y);
      lds[buf][(w * UPW + i) * 128 + lane] = x;
      lds[buf][(w * UPW + i) * 128 + 64 + lane] = y;
    }
  };
  auto stage_tail = [&](int buf, const TailScale<DT>& ts) {
    const TailValues<DT> tv(ts.down, h4, left);
#pragma unroll
    for (int i = 0; i < UPW; ++i) {
      const bool key = w * UPW + i < KU;
      const uint4* src = reinterpret_cast<const uint4*>(key ? hd.tk : hd.tv) + 2 * piece[i];
      uint4 x = src[0], y = src[1];
      if (!key) {
        x = tv.half(x, 0);
        y = tv.half(y, 1);
      }
      lds[buf][(w * UPW + i) * 128 + lane] = x;
      lds[buf][(w * UPW + i) * 128 + 64 + lane] = y;
    }
  };
  // LDS writes done, then the barrier; unlike __syncthreads() it leaves the loads of later pages in flight
  auto barrier = [&]() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto compute = [&](auto mask_tag, int buf, int pg, float cs, float v) {
    constexpr bool MASK = decltype(mask_tag)::value;
    v4f s[CT][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int c = 0; c < CT; ++c) s[c][k] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < D / 32; ++e) {
        const uint4 x = lds[buf][(k * (D / 32) + e) * 64 + lane];
#pragma unroll
        for (int c = 0; c < CT; ++c) s[c][k] = mfma<DT>(x, qv[c][e], s[c][k]);
      }
    }
    uint4 p[CT][2];
    int lim[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) lim[c] = limit[c] - pg * KV_PAGE;
    st.template softmax<MASK>(s, cs, v, lim, h4, p);
#pragma unroll
    for (int d = 0; d < D / 16; ++d) st.add(d, lds[buf][(KU + d) * 128 + lane], lds[buf][(KU + d) * 128 + 64 + lane], p);
  };
  // pages lo..open-1 are seen whole by every row of the workgroup, open..last-1 by some in part (causal)
  const int last = min(hi, full), open = max(lo, min(last, sees(row0) / KV_PAGE));
  if (lo < last) {
    load(lo);
    stage(0);
    ks = ks1;
    vs = vs1;
    if (lo + 1 < last) load(lo + 1);
    barrier();
  }
  auto step = [&](auto mask_tag, int pg) {
    const int buf = (pg - lo) & 1;
    const float cs = ks * a.scale, v = vs;
    if (pg + 1 < last) {
      stage(buf ^ 1);  // read last before the barrier that ended the step before
      ks = ks1;
      vs = vs1;
      if (pg + 2 < last) load(pg + 2);
    }
    if (pg * KV_PAGE < seen_by_any) compute(mask_tag, buf, pg, cs, v);  // 0 for a wave past the rows
    barrier();
  };
  for (int pg = lo; pg < open; ++pg) step(std::false_type{}, pg);
  for (int pg = open; pg < last; ++pg) step(std::true_type{}, pg);
  if (full < hi) {  // the unfinished page
    const TailScale<DT> ts(a.c.tail_top[(long long)hd.slot * H + h]);
    stage_tail(0, ts);
    barrier();
    if (full * KV_PAGE < seen_by_any) compute(std::true_type{}, 0, full, a.scale, ts.vs);
  }
  if (bad && t == 0) atomicOr(a.c.status, KV_ST_PAGE);
  if (!hd.there && t == 0) atomicOr(a.c.status, KV_ST_SLOT);
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const float L = st.l[c];
    const int r = wrow + 16 * c + (lane & 15);
    if (r >= rows) continue;
    const float inv = L == 0.0f ? 0.0f : 0.5f * st.unit() / L;
    if (parts <= 1) {
      const int tok = r / a.G, hq = h * a.G + r % a.G;
      uint16_t* o = a.out + b * a.sob + hq * a.soh + tok * a.sot + 4 * h4;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) store4<DT>(o + 16 * d, mean4<DT>(st.o[c][d] * inv), a.ovec);
    } else {
      const long long at = split * all_rows + (long long)bh * a.n * a.G + r;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) *reinterpret_cast<v4f*>(a.part_o + at * D + 16 * d + 4 * h4) = mean4<DT>(st.o[c][d] * inv);
      if (h4 == 0) {
        a.part_ml[2 * at] = st.m[c];
        a.part_ml[2 * at + 1] = L;
      }
    }
  }
}

// ---- joining the splits ---------------------------------------------------------------------------------
// o = sum_s w_s o_s with w_s = 2^(m_s - M) l_s / sum_t 2^(m_t - M) l_t: the parts are outputs already, so that no sum
// passes the largest value (of bf16's 3e38, say). D / 4 lanes hold a row; SG such groups share its parts
// (SG = 1, a wave reading whole rows, from 2,048 rows on; else all 256 threads one row: 1,024 rows in 12 parts take
// 29 us with their attention so and 32 the other way, 3,200 rows 52 and 51, 8,000 rows 89 and 76).
template <int DT, int D, int SG>
__global__ __launch_bounds__(256) void k_cache_attn_join(AttendArgs a) {
  constexpr int LPR = D / 4, RPW = 256 / (LPR * SG);
  __shared__ float sm[SG][RPW], sl[SG][RPW];
  __shared__ __align__(16) v4f so[SG][RPW * LPR];
  const long long all_rows = (long long)a.B * a.c.kv_heads * a.n * a.G;
  const int lane = threadIdx.x % LPR, g = threadIdx.x / LPR % SG, rw = threadIdx.x / (LPR * SG);
  const long long row = (long long)blockIdx.x * RPW + rw;
  const int H = a.c.kv_heads, per = a.n * a.G, bh = (int)(min(row, all_rows - 1) / per), r = (int)(row - (long long)bh * per);
  const int b = bh / H, h = bh % H, tok = r / a.G;
  const int nv = a.new_lens ? min(max(a.new_lens[b], 0), a.n) : a.n;
  bool there;
  const int slot = slot_of(a.c, a.slots, b, there), len = there ? held_tokens(a.c.lens[slot], a.c.max_pages) : 0;
  const int ns = min(a.splits, cdiv(cdiv(len, KV_PAGE), a.per));
  const bool live = row < all_rows && tok < nv && ns > 1;  // one part is written by its workgroup
  const float* ml = a.part_ml + 2 * (live ? row : 0);
  const float* po = a.part_o + (live ? row : 0) * D + lane * 4;
  // the group's parts are g + SG j; lane i weighs parts j = i, i + LPR, .. and hands the weights round (a group's lanes
  // run alike, so those that it asks are there)
  const int nj = live && ns > g ? cdiv(ns - g, SG) : 0;
  const long long step = SG * all_rows;
  auto at = [&](int j) { return g * all_rows + j * step; };
  float M = LOWEST, L = 0.0f, m0 = LOWEST, l0 = 0.0f;
  if (lane < nj) {
    m0 = ml[2 * at(lane)];
    l0 = ml[2 * at(lane) + 1];
  }
  M = m0;
  for (int j = lane + LPR; j < nj; j += LPR) M = fmaxf(M, ml[2 * at(j)]);
#pragma unroll
  for (int i = 1; i < LPR; i *= 2) M = fmaxf(M, __shfl_xor(M, i, LPR));
  L = l0 * exp2f(m0 - M);
  for (int j = lane + LPR; j < nj; j += LPR) L += ml[2 * at(j) + 1] * exp2f(ml[2 * at(j)] - M);
#pragma unroll
  for (int i = 1; i < LPR; i *= 2) L += __shfl_xor(L, i, LPR);
  if constexpr (SG > 1) {
    if (lane == 0) {
      sm[g][rw] = M;
      sl[g][rw] = L;
    }
    __syncthreads();
    M = sm[0][rw];
#pragma unroll
    for (int i = 1; i < SG; ++i) M = fmaxf(M, sm[i][rw]);
    L = 0.0f;
#pragma unroll
    for (int i = 0; i < SG; ++i) L += sl[i][rw] * exp2f(sm[i][rw] - M);
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int j0 = 0; j0 < nj; j0 += LPR) {
    if (j0 && j0 + lane < nj) {
      m0 = ml[2 * at(j0 + lane)];
      l0 = ml[2 * at(j0 + lane) + 1];
    }
    const float w = j0 + lane < nj ? l0 * inv * exp2f(m0 - M) : 0.0f;
    for (int j = j0; j < min(j0 + LPR, nj); j += 4) {  // four parts at a time, their loads together
      v4f v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = j + i < nj ? *reinterpret_cast<const v4f*>(po + at(j + i) * D) : v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 4; ++i) o += v[i] * __shfl(w, j - j0 + i, LPR);
    }
  }
  if constexpr (SG > 1) {
    so[g][rw * LPR + lane] = o;
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int i = 1; i < SG; ++i) o += so[i][rw * LPR + lane];
  }
  if (!live) return;
  store4<DT>(a.out + b * a.sob + (h * a.G + r % a.G) * a.soh + tok * a.sot + lane * 4, o, a.ovec);
}

// How a call is cut: which kernel, row tiles of a (sequence, kv head), and splits of the keys.
//
// Up to 32 rows of a (sequence, kv head) go to the few-rows kernel: 32 rows of 16 heads over 21,984 tokens take 24 us so
// and 25 in the other, over 87,936 tokens 40 and 49; 24 to 32 grouped rows of 8 heads of 128 25 to 49 and 29 to 53.
// The few-rows kernel gets workgroups for half the slots (two a CU; times are of calls here): with four a CU the five special rows over 274,800 tokens take 123 us
// instead of 103, the ragged batch of 32 72 instead of 74; with one 111 instead of 102 and 61 instead of 63.
//
// Many rows: four waves a workgroup, or eight (half the widening a row) at a head of 64 where the rows fill its tiles of
// 256 about as well and the cache is long. Eight for four, us at 8,000, 21,984 and 60,000 tokens of 16 heads: 400 rows
// 41, 69, 159 for 43, 76, 177; 1,500 rows 78, 181, 459 for 84, 200, 513. At 3,000 tokens 28 for 27 and 45 for 46; where half of a
// tile is empty (257 rows) 67 and 158 for 62 and 135 at the two longest; at a head of 128, causal and grouped, 166 for 150.
struct Cut {
  int ct, nw;   // nw = 0: the few-rows kernel
  int tiles, splits, per;
};

Cut cut(const ress_kv_cache& c, int B, int Hq, int n, int most_tokens) {
  Cut k{};
  const long long rows = (long long)n * (Hq / c.kv_heads), heads = (long long)B * c.kv_heads;
  // no more than the largest table holds: a larger count, rounded up to pages, would pass 32 bits
  constexpr int MOST = ((1 << 25) - 1) * KV_PAGE;
  const int pages = cdiv(most_tokens > MOST ? MOST : most_tokens > 0 ? most_tokens : 1, KV_PAGE);
  long long slots;  // workgroups that run at once
  int least;        // pages a split has at least
  if (rows <= 32) {
    k.ct = rows <= 16 ? 1 : 2;
    k.nw = 0;
    slots = 2 * CUS;
    // Two a wave; a second part, and with it a second launch, from 32 pages on (1,500 tokens 17 us in two parts, 13 in
    // one). Four a wave: one row over 344 pages 18 us instead of 17, 32 rows 22 instead of 20, 4 sequences of 63 pages 20
    // instead of 17.
    least = pages < 32 ? 16 : 8;
  } else {
    k.ct = ROWS_CT;
    const long long tiles4 = (rows + 64 * ROWS_CT - 1) / (64 * ROWS_CT);
    k.nw = c.head_dim == 64 && pages >= 64 && (tiles4 % 2 == 0 || tiles4 > 16) ? 8 : 4;
    slots = (long long)rows_waves(c.head_dim) * CUS * 4 / k.nw;
    least = 8;
  }
  const int tile = 16 * k.ct * (k.nw ? k.nw : 1);
  k.tiles = (int)((rows + tile - 1) / tile);
  // The smallest number of splits that keeps the resident slots over 90% busy, else the best of those up to
  // four rounds; a split has at least `least` pages.
  const long long wgs = heads * k.tiles;
  const int most = pages / least < 1 ? 1 : pages / least;
  double best = 0.0;
  int s = 1;
  for (int i = 1; i <= most && wgs > 0; ++i) {
    const long long all = wgs * i, rounds = (all + slots - 1) / slots;
    if (i > 1 && rounds > 4) break;
    const double fill = (double)all / (double)(rounds * slots);
    if (fill > best + 0.01) {
      best = fill;
      s = i;
    }
    if (fill > 0.9) break;
  }
  k.per = (pages + s - 1) / s;
  k.splits = (pages + k.per - 1) / k.per;
  return k;
}

long long part_floats(const ress_kv_cache& c, int B, int Hq, int n, const Cut& k) {
  return k.splits == 1 ? 0 : (long long)k.splits * B * Hq * n * (c.head_dim + 2);
}

#define RESS_READ_ONLY_ARGS a.c.table, a.c.k_scale, a.c.v_scale, a.c.lens, a.slots, a.new_lens

template <int DT, int CODES, int D>
int launch(AttendArgs& a, const Cut& k, hipStream_t stream) {
  const long long heads = (long long)a.B * a.c.kv_heads, rows = heads * a.n * a.G;
  const bool wide = rows >= 2048;  // the join's workgroups take whole rows
  const long long join = k.splits == 1 ? 0 : wide ? (rows + 1024 / D - 1) / (1024 / D) : rows;  // 256 threads, D / 4 a row
  const long long g = k.nw == 0 ? heads * k.tiles * k.splits : (heads * k.splits + 7) / 8 * 8 * k.tiles;
  RESS_REQUIRE(launchable(g, k.nw ? 64 * k.nw : 256) && launchable(join, 256),
               "ress_kv_attend: the call needs 2^32 threads or more");
  if (k.nw == 0) {
    if (k.ct == 1)
      hipLaunchKernelGGL((k_cache_attn_few<DT, CODES, D, 1>), dim3((unsigned)g), dim3(256), 0, stream, a, RESS_READ_ONLY_ARGS);
    else
      hipLaunchKernelGGL((k_cache_attn_few<DT, CODES, D, 2>), dim3((unsigned)g), dim3(256), 0, stream, a, RESS_READ_ONLY_ARGS);
    RESS_LAUNCHED("k_cache_attn_few");
  } else {
    bool eight = false;
    if constexpr (D == 64) {
      eight = k.nw == 8;
      if (eight)
        hipLaunchKernelGGL((k_cache_attn_rows<DT, CODES, D, ROWS_CT, 8>), dim3((unsigned)g), dim3(512), 0, stream, a, RESS_READ_ONLY_ARGS);
    }
    if (!eight)
      hipLaunchKernelGGL((k_cache_attn_rows<DT, CODES, D, ROWS_CT, 4>), dim3((unsigned)g), dim3(256), 0, stream, a, RESS_READ_ONLY_ARGS);
    RESS_LAUNCHED("k_cache_attn_rows");
  }
  if (k.splits > 1) {
    if (wide)
      hipLaunchKernelGGL((k_cache_attn_join<DT, D, 1>), dim3((unsigned)join), dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((k_cache_attn_join<DT, D, 256 / (D / 4)>), dim3((unsigned)join), dim3(256), 0, stream, a);
    RESS_LAUNCHED("k_cache_attn_join");
  }
  return 0;
}

}  // namespace

RESS_API long long ress_kv_attend_workspace_size(const ress_kv_cache* cache, int B, int Hq, int n, int most_tokens) {
  if (!cache || cache->kv_heads <= 0 || B < 0 || n < 0 || Hq <= 0 || Hq % cache->kv_heads) return -1;
  return 4 * part_floats(*cache, B, Hq, n, cut(*cache, B, Hq, n, most_tokens));
}

RESS_API int ress_kv_attend(const ress_kv_cache* cache, const void* q, long long sqB, long long sqH, long long sqT,
                            int B, int Hq, int n, const int* slots, const int* new_lens, int causal, float sm_scale,
                            int most_tokens, void* out, long long soB, long long soH, long long soT, void* workspace,
                            long long workspace_bytes, hipStream_t stream) {
  if (int rc = ress_kv_check(cache, B, "ress_kv_attend")) return rc;
  RESS_REQUIRE(Hq > 0 && Hq % cache->kv_heads == 0, "ress_kv_attend: %d query heads are no multiple of the cache's %d",
               Hq, cache->kv_heads);
  RESS_REQUIRE(n >= 0 && (long long)B * Hq * n < (1ll << 31), "ress_kv_attend: bad row count");
  RESS_REQUIRE(sm_scale > 0.0f && sm_scale < __builtin_huge_valf(), "ress_kv_attend: the scale must be positive and finite");
  if (B == 0 || n == 0) return 0;
  RESS_REQUIRE(q && out, "ress_kv_attend: null queries or output");
  const Cut k = cut(*cache, B, Hq, n, most_tokens);
  const long long need = part_floats(*cache, B, Hq, n, k);
  RESS_REQUIRE(workspace_bytes >= 4 * need && (need == 0 || (workspace && (uintptr_t)workspace % 16 == 0)),
               "ress_kv_attend: the workspace needs %lld bytes, 16-byte aligned", 4 * need);
  AttendArgs a{};
  a.c = *cache;
  a.q = (const uint16_t*)q; a.out = (uint16_t*)out;
  a.sqb = sqB; a.sqh = sqH; a.sqt = sqT; a.sob = soB; a.soh = soH; a.sot = soT;
  a.B = B; a.Hq = Hq; a.n = n; a.G = Hq / cache->kv_heads;
  a.slots = slots; a.new_lens = new_lens; a.causal = causal ? 1 : 0;
  a.scale = sm_scale * 1.4426950408889634f;
  a.splits = k.splits; a.per = k.per; a.tiles = k.tiles;
  a.part_o = (float*)workspace;
  a.part_ml = need ? a.part_o + (long long)k.splits * B * Hq * n * cache->head_dim : nullptr;
  a.qvec = (uintptr_t)q % 16 == 0 && sqB % 8 == 0 && sqH % 8 == 0 && sqT % 8 == 0;
  a.ovec = (uintptr_t)out % 8 == 0 && soB % 4 == 0 && soH % 4 == 0 && soT % 4 == 0;
  const bool f16 = a.c.dtype == KV_F16, fp8 = a.c.codes == KV_FP8;
  if (a.c.head_dim == 64) {
    if (f16) return fp8 ? launch<KV_F16, KV_FP8, 64>(a, k, stream) : launch<KV_F16, KV_I8, 64>(a, k, stream);
    return fp8 ? launch<KV_BF16, KV_FP8, 64>(a, k, stream) : launch<KV_BF16, KV_I8, 64>(a, k, stream);
  }
  if (f16) return fp8 ? launch<KV_F16, KV_FP8, 128>(a, k, stream) : launch<KV_F16, KV_I8, 128>(a, k, stream);
  return fp8 ? launch<KV_BF16, KV_FP8, 128>(a, k, stream) : launch<KV_BF16, KV_I8, 128>(a, k, stream);
}
