// Linear layer in 8-bit integers with a scale for each token and each output channel:
//   a_m = max_k |x_mk|, c_mk = rne(x_mk * min(127 / a_m, FLT_MAX)), s_m = a_m * fl(1/127)
//   y_mn = act((sum_k c_mk w_nk * t_n) * s_m + b_n)
// with w int8 [N][K] and t its channels' scales. The sum is exact (int32); the rest is fp32, rounded once to
// the activations' 16-bit type. A token with an element that is not finite has scale NaN, so its row of y is NaN.
//
// v_mfma_i32_16x16x64_i8 with the weights as the A operand (16 channels) and the tokens as B: a lane ends with four
// channels of one token.
#include "kvcache.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int ACT_NONE = 0, ACT_GELU = 1;
constexpr int KALIGN = 256;  // token codes are padded to this with zeros, so a product's last steps need no mask

struct Out {
  uint16_t* p;
  long long stride;
  const float *ws, *bias;
  int M, N, act;
  bool vec;  // rows are 8-byte aligned and N a multiple of 4
};

// x Phi(x). Phi(-z) = erfc(z / sqrt 2) / 2 for z >= 0 by the rational approximation 7.1.26 of Abramowitz and Stegun,
// erfc(u) = (a1 t + .. + a5 t^5) e^(-u^2), t = 1 / (1 + p u), within 1.5e-7: an absolute error of |x| 2^-23 beside
// outputs of 8 or 11 bits, in a quarter of erff's instructions (they take 8 us of a product of 1374 x 1024 x 4096).
__device__ __forceinline__ float gelu(float x) {
  const float u = fabsf(x) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, u, 1.0f));
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float half_erfc = 0.5f * (p * t) * __builtin_amdgcn_exp2f(u * u * -1.4426950408889634f);
  return x * (x < 0.0f ? half_erfc : 1.0f - half_erfc);  // NaN: t is NaN
}

// four channels n.. of token m from their sums
template <int DT>
__device__ __forceinline__ void finish4(const Out& o, int m, int n, const v4i& acc, float sx, const float (&ws)[4],
                                        const float (&bias)[4]) {
  uint16_t e[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float y = (float)acc[r] * ws[r] * sx;  // the weights' scale first: a token's may be near fp32's end, as bf16's is
    if (o.bias) y = y + bias[r];
    if (o.act == ACT_GELU) y = gelu(y);
    e[r] = Elem<DT>::put(y);
  }
  uint16_t* p = o.p + m * o.stride + n;
  if (o.vec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(e[0] | ((uint32_t)e[1] << 16), e[2] | ((uint32_t)e[3] << 16));
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < o.N) p[r] = e[r];
  }
}

__device__ __forceinline__ uint32_t top16(const uint4& v, uint32_t m) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
  return m;
}
template <int DT>
__device__ __forceinline__ uint2 codes8(const uint4& v, float inv) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = Elem<DT>::get(elem8(v, i)) * inv;
  return make_uint2(narrow4<KV_I8>(y[0], y[1], y[2], y[3]), narrow4<KV_I8>(y[4], y[5], y[6], y[7]));
}
// a row's scale and the factor its elements are multiplied by, from the bits of its largest magnitude
template <int DT>
__device__ __forceinline__ void row_scale(uint32_t top, float& scale, float& inv) {
  const float a = Elem<DT>::get((uint16_t)top);
  const bool bad = top >= Elem<DT>::INF;
  inv = bad || a == 0.0f ? 0.0f : fminf(127.0f / a, 0x1.fffffep127f);
  scale = bad ? __uint_as_float(0x7fc00000u) : a * (1.0f / 127.0f);
}

// One wave a row of K elements (a multiple of 8) -> codes [M][kp], zeros from K on, and scales. The row is held
// in registers up to 4096 elements and read again beyond. Bound by memory: 21,984 rows of 4,096 take 43 us for 270 MB
// (6.3 TB/s), 1,374 rows of 1,024 4.6 us. It is a kernel of its own because every column of the product's tiles needs the
// codes: 16 rows' maximum and codes formed in the product's loads would be formed again by each of them.
template <int DT>
__global__ __launch_bounds__(256) void k_quantize_rows(const uint16_t* __restrict__ x, long long stride, int M, int K,
                                                       uint8_t* __restrict__ codes, long long kp,
                                                       float* __restrict__ scale, bool vec) {
  constexpr int HELD = 8;  // chunks of 512 elements
  const int m = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (m >= M) return;
  const uint16_t* row = x + m * stride;
  uint4 v[HELD];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int k = i * 512 + lane * 8;
    v[i] = k < K ? ld8(row + k, vec) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < HELD; ++i) top = top16(v[i], top);
  for (int k = HELD * 512 + lane * 8; k < K; k += 512) top = top16(ld8(row + k, vec), top);
  float s, inv;
  row_scale<DT>(wave_max_u32(top), s, inv);
  uint8_t* out = codes + m * kp;
  // 0 * inf is no code: a row that is not finite has inv = 0 and its codes are forced to zero
  const bool bad = s != s;
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int k = i * 512 + lane * 8;
    if (k < kp) *reinterpret_cast<uint2*>(out + k) = bad ? make_uint2(0, 0) : codes8<DT>(v[i], inv);
  }
  for (int k = HELD * 512 + lane * 8; k < kp; k += 512)
    *reinterpret_cast<uint2*>(out + k) = bad || k >= K ? make_uint2(0, 0) : codes8<DT>(ld8(row + k, vec), inv);
  if (lane == 0) scale[m] = s;
}

// ---- many tokens: LDS-tiled product ---------------------------------------------------------------------
// A buffer of `bytes` bytes at `base` (wave-uniform) as the four words of its descriptor: reads past the end give zero.
__device__ __forceinline__ v4i descriptor(const void* base, unsigned bytes) {
  const unsigned long long p = (unsigned long long)base;
  return v4i{(int)(unsigned)p, (int)(unsigned)(p >> 32), (int)bytes, 0x00020000};
}
// 16 bytes a lane from the buffer at off + soff into LDS at lds + 16 lane. Written as assembly because the compiler,
// which does not know what the explicit waits below cover, waits for every DMA in flight before an LDS read of a
// stage that one has filled; nothing here has an output register, and m0 is set in the same block.
__device__ __forceinline__ unsigned lds_address(void* p) {
  return (unsigned)(unsigned long long)(__attribute__((address_space(3))) void*)p;
}
__device__ __forceinline__ void dma16(const v4i& rsrc, unsigned off, int soff, unsigned lds) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, %3 offen lds"
      :
      : "s"(lds), "v"(off), "s"(rsrc), "s"(soff)
      : "memory", "m0");
}
// Every DMA of the wave has landed and its LDS reads are done, then the workgroup's.
__device__ __forceinline__ void dma_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// BM tokens x BN channels a workgroup of GM x GN waves, 128 bytes of K a step in two halves, two LDS stages filled by
// DMA. A row's eight 16-byte chunks lie at place chunk ^ (row & 7), so the operand reads (16 rows, one chunk) meet no
// bank twice. A step is
//   multiply half 0, reading half 1 | its reads done and the next stage landed, barrier
//   multiply half 1, reading half 0 of the next stage, the stage just read being filled for the step after
// so there is one barrier a step, and a DMA has a whole step to land. The reads and DMAs go between the products of a
// row of tiles, a few at a time: in one run they would hold up the products behind them. A token operand is read into
// the registers of the one just used.
//
// Bound by waiting: the waves wait for half of their cycles (51%) while no unit is busy for more than a third of the launch
// (21,984 tokens, 4,096 -> 1,024: matrix cores 34%, its rounds of 464 tiles on 256 CUs included, vector 15%, LDS 14%, no
// conflicts, waits for LDS 2%). A stage's DMAs go out in one half and are waited for, all of them, after the next. 98 to 110 us
// there on different cards, 1.7 to 1.9 POP/s of the 3.9 that the matrix cores reach; 4,096 cubed 66 us, 2.1 POP/s. 1,374
// tokens, 1,024 -> 4,096, take 17 us, half of it the first fill and the epilogue. Measured against this form: four stages of 64 bytes with fewer tiles in flight, rows padded instead of swapped
// and channels permuted for wider stores, all slower; the DMA as the compiler's builtin (which waits for all of them) 151
// us for 102.
template <int DT, int BM, int BN, int GM, int GN, bool EVEN>
__global__ __launch_bounds__(64 * GM * GN, 2) void k_int8_gemm(const uint8_t* __restrict__ x, int kp,
                                                            const float* __restrict__ sx, const uint8_t* __restrict__ w,
                                                            int K, Out o) {
  constexpr int NW = GM * GN, WM = BM / GM, WN = BN / GN, TM = WM / 16, TN = WN / 16;
  constexpr int XD = BM / 8 / NW, WD = BN / 8 / NW;  // 1 KB DMAs of a wave and step, eight rows each
  static_assert(XD * 8 * NW == BM && WD * 8 * NW == BN, "every wave has whole DMAs");
  __shared__ __align__(16) uint8_t s0[(BM + BN) * 128], s1[(BM + BN) * 128];
  const int t = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, h4 = lane >> 4, r16 = lane & 15;
  // an XCD takes consecutive tiles, and these run down eight rows of tiles before they go on to the next channels:
  // what its workgroups read at one time is about square
  const int tn = cdiv(o.N, BN), total = cdiv(o.M, BM) * tn, per = cdiv(total, 8);
  const int lin = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || lin >= total) return;
  const int tm = cdiv(o.M, BM), group = lin / (8 * tn), gm = min(8, tm - 8 * group), in = lin - group * 8 * tn;
  const int m0 = (8 * group + in % gm) * BM, n0 = in / gm * BN;
  const int nrows = min(BN, o.N - n0);
  const v4i xr = descriptor(x + (long long)m0 * kp, (unsigned)(BM * kp));
  const v4i wr = descriptor(w + (long long)n0 * K, (unsigned)(nrows * K));
  // The workspace holds whole tiles of tokens (what lies past the last is multiplied, never stored). Channels past the
  // end repeat the last; chunks past a channel's row are the next one's or, past the buffer, zero: the token codes there
  // are zero.
  const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;
  const unsigned xo = (unsigned)((wv * XD * 8 + (lane >> 3)) * kp + chunk);
  unsigned wo[WD];
#pragma unroll
  for (int i = 0; i < WD; ++i) wo[i] = (unsigned)(min((wv * WD + i) * 8 + (lane >> 3), nrows - 1) * K + chunk);
  // DMA i of the wave's XD + WD
  auto fetch = [&](unsigned s, int k, int i) {
    if (i < XD) {
      dma16(xr, xo, k + i * 8 * kp, s + (wv * XD + i) * 1024);
    } else {
      // EVEN: K is a multiple of 256. Else k goes into the offset that is checked: the last channel's chunks past K lie
      // outside the buffer (an addition more a DMA, for which the largest tile has no registers left)
      const unsigned off = wo[i < XD ? 0 : i - XD];
      dma16(wr, EVEN ? off : off + k, EVEN ? k : 0, s + BM * 128 + (wv * WD + i - XD) * 1024);
    }
  };
  const int wm = wv / GN * WM, wn = wv % GN * WN;
  v4i acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = v4i{0, 0, 0, 0};
  v4i fa[2][TN], fb[TM];  // channels' operands of this half and the next, tokens' operands
  const int rd0 = r16 * 128 + (h4 ^ (r16 & 7)) * 16, rd1 = r16 * 128 + ((4 + h4) ^ (r16 & 7)) * 16;
  auto read_a = [&](const uint8_t* s, int c, int j) {
    return *reinterpret_cast<const v4i*>(s + (BM + wn + 16 * j) * 128 + (c ? rd1 : rd0));
  };
  auto read_b = [&](const uint8_t* s, int c, int i) {
    return *reinterpret_cast<const v4i*>(s + (wm + 16 * i) * 128 + (c ? rd1 : rd0));
  };
  // multiply half h; READ: the operands of half rd of stage s; FETCH: the DMAs of a stage at `at`, step k
  auto half = [&](auto h_tag, auto read_tag, auto fetch_tag, const uint8_t* s, int rd, unsigned at, int k) {
    constexpr int h = decltype(h_tag)::value;
    constexpr bool READ = decltype(read_tag)::value, FETCH = decltype(fetch_tag)::value;
    constexpr int AR = (TN + TM - 1) / TM, DR = (XD + WD + TM - 1) / TM;  // channel reads and DMAs a row of tiles
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[h][j], fb[i], acc[i][j], 0, 0, 0);
      if constexpr (READ) {
        fb[i] = read_b(s, rd, i);
#pragma unroll
        for (int j = i * AR; j < i * AR + AR; ++j)
          if (j < TN) fa[h ^ 1][j] = read_a(s, rd, j);
      }
      if constexpr (FETCH) {
#pragma unroll
        for (int d = i * DR; d < i * DR + DR; ++d)
          if (d < XD + WD) fetch(at, k, d);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const unsigned at0 = __builtin_amdgcn_readfirstlane(lds_address(s0)), at1 = __builtin_amdgcn_readfirstlane(lds_address(s1));
  const int steps = (int)(kp / 128);  // even
  constexpr std::integral_constant<int, 0> first{};
  constexpr std::integral_constant<int, 1> second{};
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
#pragma unroll
  for (int d = 0; d < XD + WD; ++d) fetch(at0, 0, d);
  dma_barrier();
#pragma unroll
  for (int d = 0; d < XD + WD; ++d) fetch(at1, 128, d);
#pragma unroll
  for (int j = 0; j < TN; ++j) fa[0][j] = read_a(s0, 0, j);
#pragma unroll
  for (int i = 0; i < TM; ++i) fb[i] = read_b(s0, 0, i);
  for (int i = 0; i + 2 < steps; i += 2) {
    half(first, yes, no, s0, 1, 0, 0);
    dma_barrier();
    half(second, yes, yes, s1, 0, at0, (i + 2) * 128);
    half(first, yes, no, s1, 1, 0, 0);
    dma_barrier();
    half(second, yes, yes, s0, 0, at1, (i + 3) * 128);
  }
  half(first, yes, no, s0, 1, 0, 0);
  dma_barrier();
  half(second, yes, no, s1, 0, 0, 0);
  half(first, yes, no, s1, 1, 0, 0);
  half(second, no, no, s1, 0, 0, 0);
  float sm[TM];  // loaded together: one at a time each store would wait for its own
#pragma unroll
  for (int i = 0; i < TM; ++i) sm[i] = sx[min(m0 + wm + 16 * i + r16, o.M - 1)];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = n0 + wn + 16 * j + 4 * h4;  // the lane's four channels
    if (n >= o.N) continue;
    float ws[4], bias[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int c = min(n + r, o.N - 1);
      ws[r] = o.ws[c];
      bias[r] = o.bias ? o.bias[c] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int m = m0 + wm + 16 * i + r16;
      if (m < o.M) finish4<DT>(o, m, n, acc[i][j], sm[i], ws, bias);
    }
  }
}

// ---- few tokens: the weights are read once, nothing else counts ------------------------------------------------
// Up to 16 tokens, 16 channels a workgroup; its NW waves quantise the tokens into LDS (each workgroup for
// itself: one launch) and share out K, the first weights loaded before. Bound by latency: one token, 1,024 -> 4,096, 4.2
// us for 4.2 MB of weights (1 TB/s).
template <int DT, int NW>
__global__ __launch_bounds__(64 * NW) void k_int8_few(const uint16_t* __restrict__ x, long long stride, int K, int kp,
                                                      const uint8_t* __restrict__ w, Out o, bool vec) {
  extern __shared__ __align__(16) uint8_t xc[];  // [M][kp]
  __shared__ float sxs[16];
  __shared__ v4i part[NW][64];
  const int t = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, h4 = lane >> 4, r16 = lane & 15;
  const int n0 = blockIdx.x * 16;
  const uint8_t* wrow = w + (long long)min(n0 + r16, o.N - 1) * K;
  const int steps = cdiv(K, 64);
  constexpr int AHEAD = 4;
  v4i a[AHEAD];
  auto fetch = [&](int s0) {  // steps s0 + i NW; 16 bytes past K (or the last step) are zero
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int k = (s0 + i * NW) * 64 + h4 * 16;
      a[i] = k < K ? *reinterpret_cast<const v4i*>(wrow + k) : v4i{0, 0, 0, 0};
    }
  };
  fetch(wv);
  float ws[4], bias[4];  // of the epilogue, loaded ahead like the weights
  if (wv == 0) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int c = min(n0 + 4 * h4 + r, o.N - 1);
      ws[r] = o.ws[c];
      bias[r] = o.bias ? o.bias[c] : 0.0f;
    }
  }
  for (int m = wv; m < o.M; m += NW) {
    const uint16_t* row = x + m * stride;
    uint32_t top = 0;
    for (int k = lane * 8; k < K; k += 512) top = top16(ld8(row + k, vec), top);
    float s, inv;
    row_scale<DT>(wave_max_u32(top), s, inv);
    for (int k = lane * 8; k < kp; k += 512)
      *reinterpret_cast<uint2*>(xc + m * kp + k) = s != s || k >= K ? make_uint2(0, 0) : codes8<DT>(ld8(row + k, vec), inv);
    if (lane == 0) sxs[m] = s;
  }
  __syncthreads();
  v4i acc = {0, 0, 0, 0};
  const uint8_t* brow = xc + min(r16, o.M - 1) * kp + h4 * 16;  // columns past the last token repeat it
  for (int s = wv; s < steps; s += AHEAD * NW) {
    v4i c[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) c[i] = a[i];
    if (s + AHEAD * NW < steps) fetch(s + AHEAD * NW);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (s + i * NW >= steps) break;
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(c[i], *reinterpret_cast<const v4i*>(brow + (s + i * NW) * 64), acc, 0, 0, 0);
    }
  }
  part[wv][lane] = acc;
  __syncthreads();
  if (wv == 0 && r16 < o.M && n0 + 4 * h4 < o.N) {
#pragma unroll
    for (int i = 1; i < NW; ++i) acc += part[i][lane];
    finish4<DT>(o, r16, n0 + 4 * h4, acc, sxs[r16], ws, bias);
  }
}

constexpr int FEW = 16, FEW_BYTES = 40 * 1024;
long long padded(int K) { return (K + KALIGN - 1) / KALIGN * (long long)KALIGN; }
// Bytes of the token codes in the workspace: whole rows of the largest tiles (192 and 256 tokens).
long long code_bytes(int M, int K) { return ((M + 255ll) / 256 * 256 + 192) * padded(K); }
bool few(int M, int K) { return M <= FEW && M * padded(K) <= FEW_BYTES; }

template <int DT>
int quantize(const void* x, long long stride, int M, int K, void* codes, long long kp, float* scale, hipStream_t stream) {
  const bool vec = (uintptr_t)x % 16 == 0 && stride % 8 == 0;
  constexpr int MOST = 1 << 25;  // rows of a launch, of 64 threads each
  for (long long m = 0; m < M; m += MOST) {
    const int rows = (int)(M - m < MOST ? M - m : MOST);
    hipLaunchKernelGGL(k_quantize_rows<DT>, dim3((rows + 3) / 4), dim3(256), 0, stream, (const uint16_t*)x + m * stride, stride,
                       rows, K, (uint8_t*)codes + m * kp, kp, scale + m, vec);
    RESS_LAUNCHED("k_quantize_rows");
  }
  return 0;
}

template <int DT, int BM, int BN, int GM, int GN>
int gemm(const uint8_t* codes, int kp, const float* sx, const void* w, int K, const Out& o, hipStream_t stream) {
  const int grid = (int)(((long long)cdiv(o.M, BM) * cdiv(o.N, BN) + 7) / 8 * 8);  // launchable: linear()
  if (K == kp)
    hipLaunchKernelGGL((k_int8_gemm<DT, BM, BN, GM, GN, true>), dim3(grid), dim3(64 * GM * GN), 0, stream, codes, kp, sx,
                       (const uint8_t*)w, K, o);
  else
    hipLaunchKernelGGL((k_int8_gemm<DT, BM, BN, GM, GN, false>), dim3(grid), dim3(64 * GM * GN), 0, stream, codes, kp, sx,
                       (const uint8_t*)w, K, o);
  RESS_LAUNCHED("k_int8_gemm");
  return 0;
}

// The tile of a product: the one whose rounds of workgroups add up to the least time. A step (128 of K) takes `alone` us
// where each CU has one tile and `full` where every CU holds the `held` that fit; a round's start and end (the output
// is written then) take `ends`. The present kernel, us of the product (256 x 256, 192 x 256, 128 x 128 | taken):
//   4096 x 4096 x 4096 66, 87, 72 | 66        21984 x 1024 (N) x 4096 (K) 107, 98, 99 | 98
//   8192 x 8192 x 8192 527, 511, 559 | 527    21984 x 4096 (N) x 1024 (K) 145, 149, 129 | 129
// and 1374 x 1024 (N) x 4096 (K): 128 x 128 24, 64 x 128 22, 64 x 64 18 | 18.
constexpr struct {
  int bm, bn, threads, held;
  double alone, full, ends;
} tiles[] = {{256, 256, 512, 1, 1.20, 1.75, 10.0}, {192, 256, 512, 1, 0.97, 1.30, 8.5}, {128, 128, 512, 2, 0.52, 1.06, 3.7},
             {64, 128, 256, 3, 0.47, 0.92, 2.5}, {64, 64, 256, 5, 0.37, 0.95, 2.0}};
int pick(int M, int N, int steps) {
  int best = 0;
  double least = 0.0;
  for (int i = 0; i < 5; ++i) {
    const double slots = 256.0 * tiles[i].held, n = (double)cdiv(M, tiles[i].bm) * cdiv(N, tiles[i].bn);
    const double rounds = floor(n / slots), rest = n / slots - rounds;
    double t = rounds * (steps * tiles[i].full + tiles[i].ends);
    if (rest > 0.0) t += steps * fmax(tiles[i].alone, rest * tiles[i].full) + 0.6 * tiles[i].ends;
    if (i == 0 || t < least) {
      least = t;
      best = i;
    }
  }
  return best;
}

template <int DT>
int linear(const void* x, long long stride, int K, const void* w, const Out& o, void* workspace, hipStream_t stream) {
  const long long kp = padded(K);
  if (few(o.M, K)) {
    const bool vec = (uintptr_t)x % 16 == 0 && stride % 8 == 0;
    const dim3 grid(cdiv(o.N, 16));
    if (grid.x >= 128)
      hipLaunchKernelGGL((k_int8_few<DT, 4>), grid, dim3(256), o.M * kp, stream, (const uint16_t*)x, stride, K, (int)kp,
                         (const uint8_t*)w, o, vec);
    else
      hipLaunchKernelGGL((k_int8_few<DT, 16>), grid, dim3(1024), o.M * kp, stream, (const uint16_t*)x, stride, K, (int)kp,
                         (const uint8_t*)w, o, vec);
    RESS_LAUNCHED("k_int8_few");
    return 0;
  }
  const int tile = pick(o.M, o.N, (int)(kp / 128));
  RESS_REQUIRE(launchable((long long)cdiv(o.M, tiles[tile].bm) * cdiv(o.N, tiles[tile].bn) + 7, tiles[tile].threads),
               "ress_int8_linear: the call needs 2^32 threads or more");
  uint8_t* codes = (uint8_t*)workspace;
  float* sx = (float*)(codes + code_bytes(o.M, K));
  if (int rc = quantize<DT>(x, stride, o.M, K, codes, kp, sx, stream)) return rc;
  switch (tile) {
    case 0: return gemm<DT, 256, 256, 2, 4>(codes, (int)kp, sx, w, K, o, stream);
    case 1: return gemm<DT, 192, 256, 2, 4>(codes, (int)kp, sx, w, K, o, stream);
    case 2: return gemm<DT, 128, 128, 2, 4>(codes, (int)kp, sx, w, K, o, stream);
    case 3: return gemm<DT, 64, 128, 2, 2>(codes, (int)kp, sx, w, K, o, stream);
    default: return gemm<DT, 64, 64, 2, 2>(codes, (int)kp, sx, w, K, o, stream);
  }
}

int check_rows(const char* who, int dtype, int M, int K) {
  RESS_REQUIRE(dtype == KV_BF16 || dtype == KV_F16, "%s: dtype code %d is not 1 (bf16) or 2 (fp16)", who, dtype);
  RESS_REQUIRE(M >= 0 && M <= (1 << 30) && K >= 0 && K % 16 == 0 && K <= 131072, "%s: %d rows of %d elements (a multiple of 16, at most 131072; at most 2^30 rows)",
               who, M, K);
  return 0;
}

}  // namespace

RESS_API int ress_quantize_rows(const void* x, long long stride, int dtype, int M, int K, void* codes,
                                long long code_stride, float* scale, hipStream_t stream) {
  if (int rc = check_rows("ress_quantize_rows", dtype, M, K)) return rc;
  if (M == 0) return 0;
  RESS_REQUIRE(K > 0, "ress_quantize_rows: rows without elements");
  RESS_REQUIRE(x && codes && scale, "ress_quantize_rows: null pointer");
  RESS_REQUIRE((uintptr_t)codes % 8 == 0 && code_stride % 8 == 0 && code_stride >= K,
               "ress_quantize_rows: codes must be 8-byte aligned rows of at least %d bytes", K);
  return dtype == KV_BF16 ? quantize<KV_BF16>(x, stride, M, K, codes, code_stride, scale, stream)
                          : quantize<KV_F16>(x, stride, M, K, codes, code_stride, scale, stream);
}

RESS_API long long ress_int8_linear_workspace_size(int M, int K, int N) {
  if (M < 0 || K < 0 || N < 0) return -1;
  return few(M, K) ? 0 : code_bytes(M, K) + 4ll * M;
}

RESS_API int ress_int8_linear_tile(int M, int K, int N) {
  if (M <= 0 || K <= 0 || N <= 0 || few(M, K)) return 0;
  const auto& t = tiles[pick(M, N, (int)(padded(K) / 128))];
  return t.bm << 16 | t.bn;
}

RESS_API int ress_int8_linear(const void* x, long long stride, int dtype, int M, int K, int N, const void* w,
                              const float* w_scale, const float* bias, int act, void* out, long long out_stride,
                              void* workspace, long long workspace_bytes, hipStream_t stream) {
  if (int rc = check_rows("ress_int8_linear", dtype, M, K)) return rc;
  RESS_REQUIRE(N >= 0 && N <= (1 << 24), "ress_int8_linear: bad channel count %d", N);
  RESS_REQUIRE(act == ACT_NONE || act == ACT_GELU, "ress_int8_linear: act %d is not 0 (none) or 1 (gelu)", act);
  if (M == 0 || N == 0) return 0;
  RESS_REQUIRE(K > 0, "ress_int8_linear: rows without elements");
  RESS_REQUIRE(x && w && w_scale && out, "ress_int8_linear: null pointer");
  RESS_REQUIRE((uintptr_t)w % 16 == 0, "ress_int8_linear: the weights are not 16-byte aligned");
  const long long need = ress_int8_linear_workspace_size(M, K, N);
  RESS_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && (uintptr_t)workspace % 16 == 0)),
               "ress_int8_linear: the workspace needs %lld bytes, 16-byte aligned", need);
  const Out o{(uint16_t*)out, out_stride, w_scale, bias, M, N, act,
              (uintptr_t)out % 8 == 0 && out_stride % 4 == 0 && N % 4 == 0};
  return dtype == KV_BF16 ? linear<KV_BF16>(x, stride, K, w, o, workspace, stream)
                          : linear<KV_F16>(x, stride, K, w, o, workspace, stream);
}
