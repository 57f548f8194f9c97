// Linear layer in 8-bit integers with a scale for each token and each output channel:
//   a_m = max_k |x_mk|, c_mk = rne(x_mk * min(127 / a_m, FLT_MAX)), s_m = a_m * fl(1/127)
//   y_mn = act((s_m * sum_k c_mk w_nk) * t_n + b_n)
// with w int8 [N][K] and t its channels' scales. The sum is exact (int32); the rest is fp32, rounded once to
// the activations' 16-bit type. A token with an element that is not finite has scale NaN, so its row of y is NaN.
//
// v_mfma_i32_16x16x64_i8 with the weights as the A operand (16 channels) and the tokens as B: a lane ends with
// four consecutive channels of one token, one 8-byte store.
#include "kvcache.h"

#ifndef RESS_GEMM
#define RESS_GEMM 128, 128, 2, 2, 2
#endif

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int ACT_NONE = 0, ACT_GELU = 1;
constexpr int KALIGN = 128;  // token codes are padded to this with zeros, so a product's last step needs no mask

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
    float y = (float)acc[r] * sx * ws[r];
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
// in registers up to 4096 elements and read again beyond.
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
#define RESS_I8_DWORD3 0x00020000
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rsrc, unsigned voffset, int soffset, void* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)lds, 16, (int)voffset, soffset,
                                           0, 0);
}
// Waits until at most N of the wave's DMAs are in flight, then for the workgroup. __syncthreads() would wait for
// all of them.
template <int N>
__device__ __forceinline__ void dma_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// BM tokens x BN channels a workgroup of GM x GN waves, 128 bytes of K a step, LDS stages filled by DMA ahead of
// their use (STAGES - 1 steps). A row's eight 16-byte chunks lie at place chunk ^ (row & 7), so the operand reads
// (16 rows, one chunk) meet no bank twice.
template <int DT, int BM, int BN, int GM, int GN, int STAGES>
__global__ __launch_bounds__(64 * GM * GN) void k_int8_gemm(const uint8_t* __restrict__ x, long long kp,
                                                            const float* __restrict__ sx, const uint8_t* __restrict__ w,
                                                            int K, Out o) {
  constexpr int NW = GM * GN, WM = BM / GM, WN = BN / GN, TM = WM / 16, TN = WN / 16;
  constexpr int ROWS = BM + BN;             // tokens, then channels
  constexpr int XD = BM / 8 / NW, WD = BN / 8 / NW;  // 1 KB DMAs of a wave: eight rows each
  static_assert(XD * 8 * NW == BM && WD * 8 * NW == BN, "every wave has whole DMAs");
  // distinct objects: the compiler sees that a DMA writes no stage that is being read
  __shared__ __align__(16) uint8_t s0[ROWS * 128], s1[ROWS * 128], s2[STAGES > 2 ? ROWS * 128 : 16];
  const int t = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63, h4 = lane >> 4, r16 = lane & 15;
  // an XCD takes consecutive tiles, channels fastest: its L2 keeps the weights, and a row of tiles its tokens
  const int tn = cdiv(o.N, BN), total = cdiv(o.M, BM) * tn, per = cdiv(total, 8);
  const int lin = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || lin >= total) return;
  const int m0 = lin / tn * BM, n0 = lin % tn * BN;
  const int mrows = min(BM, o.M - m0), nrows = min(BN, o.N - n0);
  const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(x + (long long)m0 * kp), (short)0, (int)(mrows * kp), RESS_I8_DWORD3);
  const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(w + (long long)n0 * K), (short)0, nrows * K, RESS_I8_DWORD3);
  // Rows past the end repeat the last (never stored); chunks past a channel's row repeat its last, where the token
  // codes are zero.
  unsigned xo[XD], wo[WD];
#pragma unroll
  for (int i = 0; i < XD; ++i) {
    const int row = (wv * XD + i) * 8 + (lane >> 3);
    xo[i] = (unsigned)(min(row, mrows - 1) * (int)kp + ((lane & 7) ^ (row & 7)) * 16);
  }
#pragma unroll
  for (int i = 0; i < WD; ++i) {
    const int row = (wv * WD + i) * 8 + (lane >> 3);
    wo[i] = (unsigned)(min(row, nrows - 1) * K + ((lane & 7) ^ (row & 7)) * 16);
  }
  auto fetch = [&](uint8_t* s, int k) {
#pragma unroll
    for (int i = 0; i < XD; ++i) dma16(xr, xo[i], k, s + (wv * XD + i) * 1024);
#pragma unroll
    for (int i = 0; i < WD; ++i) {
      unsigned off = wo[i];
      if (k + 128 > K) {  // the last step of a K that is no multiple of 128
        const int row = (wv * WD + i) * 8 + (lane >> 3);
        off = (unsigned)(min(row, nrows - 1) * K + min(((lane & 7) ^ (row & 7)) * 16, K - 16 - k));
      }
      dma16(wr, off, k, s + BM * 128 + (wv * WD + i) * 1024);
    }
  };
  const int wm = wv / GN * WM, wn = wv % GN * WN;
  v4i acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = v4i{0, 0, 0, 0};
  auto compute = [&](const uint8_t* s) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      v4i a[TN], b[TM];
      const int place = ((4 * k + h4) ^ (r16 & 7)) * 16;
#pragma unroll
      for (int i = 0; i < TM; ++i) b[i] = *reinterpret_cast<const v4i*>(s + (wm + 16 * i + r16) * 128 + place);
#pragma unroll
      for (int j = 0; j < TN; ++j) a[j] = *reinterpret_cast<const v4i*>(s + (BM + wn + 16 * j + r16) * 128 + place);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[j], b[i], acc[i][j], 0, 0, 0);
    }
  };
  const int steps = (int)(kp / 128);
  constexpr int DMAS = XD + WD;
  if constexpr (STAGES == 3) {
    // a step's DMA was started two steps before: the newest may stay in flight
    auto step = [&](const uint8_t* cur, uint8_t* ahead, int i) {
      if (i + 2 < steps) fetch(ahead, (i + 2) * 128);
      compute(cur);
      if (i + 2 < steps) dma_barrier<DMAS>();
      else dma_barrier<0>();
    };
    fetch(s0, 0);
    if (steps > 1) {
      fetch(s1, 128);
      dma_barrier<DMAS>();
    } else {
      dma_barrier<0>();
    }
    int i = 0;
    for (; i + 3 <= steps; i += 3) {
      step(s0, s2, i);
      step(s1, s0, i + 1);
      step(s2, s1, i + 2);
    }
    if (i < steps) step(s0, s2, i++);
    if (i < steps) step(s1, s0, i++);
  } else {
    auto step = [&](const uint8_t* cur, uint8_t* nxt, int i) {
      if (i + 1 < steps) fetch(nxt, (i + 1) * 128);
      compute(cur);
      dma_barrier<0>();
    };
    fetch(s0, 0);
    dma_barrier<0>();
    int i = 0;
    for (; i + 2 <= steps; i += 2) {
      step(s0, s1, i);
      step(s1, s0, i + 1);
    }
    if (i < steps) step(s0, s1, i);
  }
  // the epilogue's scales once per lane
  float sm[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) sm[i] = sx[min(m0 + wm + 16 * i + r16, o.M - 1)];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = n0 + wn + 16 * j + 4 * h4;
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
// itself: one launch) and share out K, the first weights loaded before.
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
bool few(int M, int K) { return M <= FEW && M * padded(K) <= FEW_BYTES; }

template <int DT>
int quantize(const void* x, long long stride, int M, int K, void* codes, long long kp, float* scale, hipStream_t stream) {
  const bool vec = (uintptr_t)x % 16 == 0 && stride % 8 == 0;
  hipLaunchKernelGGL(k_quantize_rows<DT>, dim3((M + 3) / 4), dim3(256), 0, stream, (const uint16_t*)x, stride, M, K,
                     (uint8_t*)codes, kp, scale, vec);
  RESS_LAUNCHED("k_quantize_rows");
  return 0;
}

template <int DT, int BM, int BN, int GM, int GN, int STAGES>
int gemm(const uint8_t* codes, long long kp, const float* sx, const void* w, int K, const Out& o, hipStream_t stream) {
  const long long tiles = (long long)cdiv(o.M, BM) * cdiv(o.N, BN);
  RESS_REQUIRE(tiles < (1ll << 30), "ress_int8_linear: the call needs too many workgroups");
  const int grid = (int)((tiles + 7) / 8 * 8);
  hipLaunchKernelGGL((k_int8_gemm<DT, BM, BN, GM, GN, STAGES>), dim3(grid), dim3(64 * GM * GN), 0, stream, codes, kp, sx,
                     (const uint8_t*)w, K, o);
  RESS_LAUNCHED("k_int8_gemm");
  return 0;
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
  uint8_t* codes = (uint8_t*)workspace;
  float* sx = (float*)(codes + (long long)o.M * kp);
  if (int rc = quantize<DT>(x, stride, o.M, K, codes, kp, sx, stream)) return rc;
  return gemm<DT, RESS_GEMM>(codes, kp, sx, w, K, o, stream);
}

int check_rows(const char* who, int dtype, int M, int K) {
  RESS_REQUIRE(dtype == KV_BF16 || dtype == KV_F16, "%s: dtype code %d is not 1 (bf16) or 2 (fp16)", who, dtype);
  RESS_REQUIRE(M >= 0 && K >= 0 && K % 16 == 0 && K <= 131072, "%s: %d rows of %d elements (a multiple of 16, at most 131072)",
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
  return few(M, K) ? 0 : (long long)M * padded(K) + 4ll * M;
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
