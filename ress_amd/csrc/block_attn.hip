// Softmax attention with a backward pass, over 128-query x 64-key blocks.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j - lse_i)     over the keys j that row i sees
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta),  delta_i = dO_i.o_i,  dQ = scale dS K,  dK = scale dS^T Q
//
// Row i of a sequence sees the keys below its length; causal: those up to i + k_len - q_len; with a map: those of the 64-key
// blocks that the map keeps for its 128-query block. Nothing of the probabilities is stored: the backward pass forms them
// anew from lse.
//
// All products are 32x32x16 MFMAs on 16-bit operands with fp32 sums. A lane of the result holds one column and, of each 16
// rows, four and four: {4h..4h+3, 8+4h..8+4h+3}, h its half of the wave. That is what the next product takes as its B operand
// once its A operand holds the 16 places in the same order, so P and dS go from one product's registers into the next:
//   forward, dQ:  S^T = K Q^T (column: the lane's query), O^T += V^T P^T, dP^T = V dO^T, dQ^T += K^T dS^T
//   dK and dV:    S = Q K^T (column: the lane's key), dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS
// Transposed A operands (V^T, K^T, dO^T, Q^T) come out of the row-major LDS tiles by ds_read_tr16_b64, which gives lane i of 16 the
// i-th column of a 4 x 16 block. dQ and dK/dV are kernels of their own, each the owner of its rows: S and dP are computed
// twice (18 products' worth of operations for the 14 that a step needs), and nothing is added by atomics, so results
// repeat bit for bit.
#include "../../include/ress_hip.h"
#include "block_attn.h"

namespace {

// ---- forward ----------------------------------------------------------------
template <int DT, int D, bool MAP>
__global__ __launch_bounds__(256, 2) void k_block_attn_fwd(AttnArgs a) {
  __shared__ __align__(16) uint8_t lds[2][2 * tile_bytes(D)];
  extern __shared__ uint32_t bits[];
  const Lane<D> ln;
  Item it;
  if (!it.query_tile(a)) return;
  const Head hd(a, it.b, it.h / a.G);
  const int qlen = a.q_len(it.b), q0 = it.tile * QB;
  const int w = ln.wave, row = q0 + 32 * w + ln.c32;
  v16f o[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d) o[d] = zero16();
  float m = LOWEST, l = 0.0f;
  if (q0 < qlen) {
    const int off = hd.klen - qlen;
    const int sees = a.causal ? min(hd.klen, max(0, row + off + 1)) : hd.klen;
    const int last = min(q0 + QB, qlen) - 1;
    const int most = a.causal ? min(hd.klen, max(0, last + off + 1)) : hd.klen;
    const int nfull = (a.causal ? min(hd.klen, max(0, q0 + off + 1)) : hd.klen) / KB;  // blocks that every row sees whole
    uint4 q[D / 16];
    load_row<D>(a.q, it.b, it.h, row, row < qlen, ln.half, q);
    Walk<MAP> walk(a, it, cdiv(most, KB), bits);
    const Stream<D> ks(a.k, hd.kbase(a.k), ln, 4), vs(a.v, hd.kbase(a.v), ln, 4);
    auto fetch = [&](int buf, int kb) {
      ks.fetch(lds[buf], kb * KB, hd.klen, w);
      vs.fetch(lds[buf] + tile_bytes(D), kb * KB, hd.klen, w);
    };
    run_steps(walk, fetch, [&](int buf, int kb) {
      const uint8_t* tile = lds[buf];
      v16f s[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) s[t] = rows_times<DT, D>(tile, 32 * t, ln, q, zero16());
      if (kb >= nfull) {
        const int below = sees - kb * KB - 4 * ln.half;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[t][r] = 32 * t + c_row(r) < below ? s[t][r] : -__builtin_huge_valf();
      }
      float top = LOWEST;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[t][r]);
      top = pair_max(top);
      top = top == LOWEST ? LOWEST : top * a.scale2;
      if (__any(top > m + LAZY)) {
        const float mn = top > m + LAZY ? top : m;
        const float f = exp2f(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= f;
      }
      uint4 p[2][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float e[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          e[r] = __builtin_amdgcn_exp2f(fmaf(s[t][r], a.scale2, -m));
          l += e[r];
        }
        pack16<DT>(e, p[t]);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int d = 0; d < D / 32; ++d) o[d] = columns_times<DT, D>(tile + tile_bytes(D), 32 * t, d, ln, p[t], o[d]);
    });
  }
  l = pair_sum(l);
  const bool some = row < qlen && (l > 0.0f || l != l);
  if (row < a.Tq) {
    store_out<DT, D>(a, it, row, ln.half, o, 1.0f / l, some);
    if (a.lse && ln.half == 0) a.lse[a.row_at(it, row)] = some ? m + log2f(l) : __builtin_huge_valf();
  }
}

// ---- backward: row sums -----------------------------------------------------
// -delta_i = -dO_i.(o_i + what o's rounding took), lse less the lift of P, and fp16: the largest finite |dO| of each
// (sequence, key/value head). Bound by its bytes.
template <int DT, int D>
__global__ __launch_bounds__(256) void k_block_attn_delta(AttnArgs a, int chunks) {
  constexpr int LR = D / 8;
  const int bh = blockIdx.x / chunks, b = bh / a.Hq, h = bh % a.Hq, piece = threadIdx.x % LR;
  const int from = blockIdx.x % chunks * DELTA_ROWS, end = min(a.Tq, from + DELTA_ROWS), qlen = a.q_len(b);
  float top = 0.0f;
  for (int i = from + threadIdx.x / LR; i < end; i += 256 / LR) {  // a row's lanes go together
    float sum = 0.0f;
    const long long r = (long long)bh * a.Tq + i;
    if (i < qlen) {
      float x[8], y[8], z[8];
      unpack8<DT>(*reinterpret_cast<const uint4*>(a.go.at(b, h, i) + 8 * piece), x);
      unpack8<DT>(*reinterpret_cast<const uint4*>(a.o.at(b, h, i) + 8 * piece), y);
      unpack8<DT>(*reinterpret_cast<const uint4*>(a.rest + r * D + 8 * piece), z);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        sum = fmaf(x[u], y[u] + z[u], sum);
        const float m = fabsf(x[u]);
        if (m > top && m < __builtin_huge_valf()) top = m;
      }
    }
#pragma unroll
    for (int s = 1; s < LR; s <<= 1) sum += __shfl_xor(sum, s, LR);
    if (piece == 0) {
      a.ndelta[r] = -sum;
      a.lse_b[r] = a.lse[r] - lift(DT);
    }
  }
  if constexpr (DT == BA_F16) {
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0 && top > 0.0f) atomicMax(a.top + (long long)b * a.Hk + h / a.G, __float_as_uint(top));
  }
}
__global__ void k_block_attn_clear(uint32_t* p, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) p[i] = 0;
}
// the largest finite |v| of each (sequence, key/value head), fp16
template <int D>
__global__ __launch_bounds__(256) void k_block_attn_vtop(AttnArgs a, int chunks) {
  constexpr int LR = D / 8;
  const int bh = blockIdx.x / chunks, chunk = blockIdx.x % chunks, b = bh / a.Hk, h = bh % a.Hk;
  const int end = min(a.k_len(b), (chunk + 1) * VTOP_ROWS);
  float top = 0.0f;
  for (int i = chunk * VTOP_ROWS + threadIdx.x / LR; i < end; i += 256 / LR) {
    float x[8];
    unpack8<BA_F16>(*reinterpret_cast<const uint4*>(a.v.at(b, h, i) + 8 * (threadIdx.x % LR)), x);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float m = fabsf(x[u]);
      if (m > top && m < __builtin_huge_valf()) top = m;
    }
  }
  top = wave_max(top);
  if ((threadIdx.x & 63) == 0 && top > 0.0f) atomicMax(a.top + (long long)a.B * a.Hk + bh, __float_as_uint(top));
}

// fp16: dS is formed times a power of two that takes the largest possible one to 2^15 (|dP - delta| <= 2 D max|dO| max|v|,
// P <= 1): a gradient far below fp16's smallest number keeps its bits. bf16 has fp32's range.
template <int DT, int D>
__device__ __forceinline__ float lift_ds(const AttnArgs& a, int b, int hk) {
  if constexpr (DT == BA_BF16) return 1.0f;
  const int at = b * a.Hk + hk;
  const float most = __uint_as_float(a.top[at]) * __uint_as_float(a.top[(long long)a.B * a.Hk + at]);
  if (!(most > 0.0f)) return 1.0f;
  int e;
  frexpf(most, &e);  // most < 2^e
  return ldexpf(1.0f, min(max(15 - (D == 64 ? 7 : 8) - e, -100), 100));
}

// ---- backward: dQ -----------------------------------------------------------
template <int DT, int D, bool MAP>
__global__ __launch_bounds__(256, 2) void k_block_attn_dq(AttnArgs a) {
  __shared__ __align__(16) uint8_t lds[2][2 * tile_bytes(D)];
  extern __shared__ uint32_t bits[];
  const Lane<D> ln;
  Item it;
  if (!it.query_tile(a)) return;
  const Head hd(a, it.b, it.h / a.G);
  const int qlen = a.q_len(it.b), q0 = it.tile * QB;
  const int w = ln.wave, row = q0 + 32 * w + ln.c32;
  v16f dq[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d) dq[d] = zero16();
  float undo = 0.0f;
  if (q0 < qlen) {
    const int off = hd.klen - qlen;
    const int sees = a.causal ? min(hd.klen, max(0, row + off + 1)) : hd.klen;
    const int last = min(q0 + QB, qlen) - 1;
    const int most = a.causal ? min(hd.klen, max(0, last + off + 1)) : hd.klen;
    const int nfull = (a.causal ? min(hd.klen, max(0, q0 + off + 1)) : hd.klen) / KB;
    uint4 q[D / 16], g[D / 16];
    load_row<D>(a.q, it.b, it.h, row, row < qlen, ln.half, q);
    load_row<D>(a.go, it.b, it.h, row, row < qlen, ln.half, g);
    const float f = lift_ds<DT, D>(a, it.b, it.h / a.G);
    undo = a.scale / f;
    float lse = 0.0f, nd = 0.0f;
    if (row < qlen) {
      lse = a.lse_b[a.row_at(it, row)] + lift(DT) - log2f(f);
      nd = a.ndelta[a.row_at(it, row)];
    }
    v16f ndelta;
#pragma unroll
    for (int r = 0; r < 16; ++r) ndelta[r] = nd;
    Walk<MAP> walk(a, it, cdiv(most, KB), bits);
    const Stream<D> ks(a.k, hd.kbase(a.k), ln, 4), vs(a.v, hd.kbase(a.v), ln, 4);
    auto fetch = [&](int buf, int kb) {
      ks.fetch(lds[buf], kb * KB, hd.klen, w);
      vs.fetch(lds[buf] + tile_bytes(D), kb * KB, hd.klen, w);
    };
    run_steps(walk, fetch, [&](int buf, int kb) {
      const uint8_t* tile = lds[buf];
      each<2>([&](auto t_) {
        constexpr int t = decltype(t_)::value;
        const v16f s = rows_times<DT, D>(tile, 32 * t, ln, q, zero16());
        const v16f dp = rows_times<DT, D>(tile + tile_bytes(D), 32 * t, ln, g, ndelta);
        float e[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, -lse)) * dp[r];
        if (kb >= nfull) {
          const int below = sees - kb * KB - 4 * ln.half;
#pragma unroll
          for (int r = 0; r < 16; ++r) e[r] = 32 * t + c_row(r) < below ? e[r] : 0.0f;
        }
        uint4 ds[2];
        pack16<DT>(e, ds);
        each<D / 32>([&](auto d) { dq[d] = columns_times<DT, D>(tile, 32 * t, d, ln, ds, dq[d]); });
      });
    });
  }
  if (row < a.Tq) store_grad<DT, D>(a.dq, it.b, it.h, row, ln.half, dq, undo, row < qlen);
}

// ---- backward: dK and dV ----------------------------------------------------
template <int DT, int D, int NW, bool MAP>
__global__ __launch_bounds__(64 * NW, 2) void k_block_attn_dkv(AttnArgs a) {
  constexpr int T = tile_bytes(D);
  __shared__ __align__(16) uint8_t lds[2][2 * T + 512];
  extern __shared__ uint32_t bits[];
  const Lane<D> ln;
  Item it;
  if (!it.key_tile(a, 32 * NW)) return;
  const Head hd(a, it.b, it.h);
  const int qlen = a.q_len(it.b), k0 = it.tile * 32 * NW;
  const int w = ln.wave, key = k0 + 32 * w + ln.c32;
  v16f dk[D / 32], dv[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d) dk[d] = dv[d] = zero16();
  float f = 1.0f;
  if (k0 < hd.klen && qlen > 0) {
    const int off = hd.klen - qlen;
    uint4 k[D / 16], v[D / 16];
    load_row<D>(a.k, it.b, it.h, key, key < hd.klen, ln.half, k);
    load_row<D>(a.v, it.b, it.h, key, key < hd.klen, ln.half, v);
    f = lift_ds<DT, D>(a, it.b, it.h);
    const float fp = f * (DT == BA_F16 ? 0x1p-14f : 1.0f);
    const int from = a.causal ? min(qlen, max(0, k0 - off)) : 0;          // no row before it sees a key of the tile
    const int whole = a.causal ? max(0, k0 + 32 * NW - 1 - off) : 0;      // rows from here on see all of it
    const int first = a.causal ? key - off - 4 * ln.half : 0;             // rows from `first` on see the lane's key
    for (int g = 0; g < a.G; ++g) {
      const int h = it.h * a.G + g;
      WalkColumn<MAP> walk(a, it.b, h, k0 / KB, from / QS, cdiv(qlen, QS), bits, g > 0);
      const Stream<D> qs(a.q, a.q.at(it.b, h, 0), ln, NW), gs(a.go, a.go.at(it.b, h, 0), ln, NW);
      const long long rows = ((long long)it.b * a.Hq + h) * a.Tq;
      auto fetch = [&](int buf, int st) {
        qs.fetch(lds[buf], st * QS, qlen, w);
        gs.fetch(lds[buf] + T, st * QS, qlen, w);
        if (w == 0) fetch_row_values(a.lse_b + rows + st * QS, qlen - st * QS, lds[buf] + 2 * T);
        if (w == 1) fetch_row_values(a.ndelta + rows + st * QS, qlen - st * QS, lds[buf] + 2 * T + 256);
      };
      run_steps(walk, fetch, [&](int buf, int st) {
        const uint8_t* tile = lds[buf];
        each<2>([&](auto t_) {
          constexpr int t = decltype(t_)::value;
          const v16f s = rows_times<DT, D>(tile, 32 * t, ln, k, zero16());
          const v16f lse = row_values(tile + 2 * T, 32 * t, ln);
          float e[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, -lse[r]));
          if (st * QS < whole) {
#pragma unroll
            for (int r = 0; r < 16; ++r) e[r] = st * QS + 32 * t + c_row(r) >= first ? e[r] : 0.0f;
          }
          uint4 p[2], ds[2];
          pack16<DT>(e, p);
#ifdef SB1
          if (D == 128) __builtin_amdgcn_sched_barrier(0);
#endif
          const v16f dp = rows_times<DT, D>(tile + T, 32 * t, ln, v, row_values(tile + 2 * T + 256, 32 * t, ln));
          each<D / 32>([&](auto x) { dv[x] = columns_times<DT, D>(tile + T, 32 * t, x, ln, p, dv[x]); });
#ifdef SB3
          if (D == 128) __builtin_amdgcn_sched_barrier(0);
#endif
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            e[r] *= dp[r];
            if constexpr (DT == BA_F16) e[r] *= fp;
          }
          pack16<DT>(e, ds);
          each<D / 32>([&](auto x) { dk[x] = columns_times<DT, D>(tile, 32 * t, x, ln, ds, dk[x]); });
#ifdef SB2
          __builtin_amdgcn_sched_barrier(0);
#endif
        });
      });
    }
  }
  if (key < a.Tk) {
    store_grad<DT, D>(a.dk, it.b, it.h, key, ln.half, dk, a.scale / f, key < hd.klen);
    store_grad<DT, D>(a.dv, it.b, it.h, key, ln.half, dv, DT == BA_F16 ? 0x1p-14f : 1.0f, key < hd.klen);
  }
}

// ---- host -------------------------------------------------------------------
bool fits(const View& x, int heads, int T, int D) {
  const long long lo = D, most = 1ll << 24;
  return x.p && ((uintptr_t)x.p & 15) == 0 && x.b >= 0 && x.h >= 0 && (x.b & 7) == 0 && (x.h & 7) == 0 && (x.t & 7) == 0 &&
         x.t >= lo && x.t < most;
}
int check(const AttnArgs& a, int D, int dtype, const char* name) {
  RESS_REQUIRE(D == 64 || D == 128, "%s: head_dim %d (64 or 128)", name, D);
  RESS_REQUIRE(dtype == BA_BF16 || dtype == BA_F16, "%s: dtype code %d", name, dtype);
  RESS_REQUIRE(a.B >= 0 && a.Hq >= 0 && a.Hk >= 1 && a.Tq >= 0 && a.Tk >= 0 && a.Hq % a.Hk == 0, "%s: bad geometry", name);
  RESS_REQUIRE(a.Tq <= 1 << 26 && a.Tk <= 1 << 26, "%s: more than 2^26 tokens", name);
  RESS_REQUIRE(!a.map || (a.Tq <= 1 << 20 && a.Tk <= 1 << 20), "%s: more than 2^20 tokens under a map", name);
  RESS_REQUIRE(a.scale > 0.0f && a.scale < __builtin_inff(), "%s: scale must be positive and finite", name);
  return 0;
}
int grid(long long items, int threads, const char* name, unsigned* blocks) {
  const long long n = (items + 7) / 8 * 8;
  RESS_REQUIRE(n * threads < 1ll << 32, "%s: 2^32 threads or more", name);
  *blocks = (unsigned)n;
  return 0;
}
size_t bit_bytes(int n) { return 8 * (size_t)cdiv(n, 64); }

#define RESS_BA_CASE(DT_, D_, ...)        \
  if (dtype == DT_ && D == D_) {          \
    constexpr int DT = DT_, DIM = D_;     \
    __VA_ARGS__                           \
  }
#define RESS_BA_EACH(...)                 \
  RESS_BA_CASE(BA_BF16, 64, __VA_ARGS__)  \
  RESS_BA_CASE(BA_BF16, 128, __VA_ARGS__) \
  RESS_BA_CASE(BA_F16, 64, __VA_ARGS__)   \
  RESS_BA_CASE(BA_F16, 128, __VA_ARGS__)

View view(const ress_strided& x) { return View{(uint16_t*)x.data, x.sb, x.sh, x.st}; }

AttnArgs arguments(const ress_block_attn* c) {
  AttnArgs a{};
  a.q = view(c->q);
  a.k = view(c->k);
  a.v = view(c->v);
  a.o = view(c->out);
  a.B = c->B;
  a.Hq = c->q_heads;
  a.Hk = c->kv_heads;
  a.G = c->kv_heads > 0 ? c->q_heads / c->kv_heads : 0;
  a.Tq = c->Tq;
  a.Tk = c->Tk;
  a.q_lens = c->q_lens;
  a.k_lens = c->k_lens;
  a.map = (const uint8_t*)c->map;
  a.mb = c->map_sb;
  a.mh = c->map_sh;
  a.mq = c->map_sq;
  a.mk = c->map_sk;
  a.causal = c->causal;
  a.scale = c->scale;
  a.scale2 = c->scale * 1.44269504088896340736f;
  a.rest = (uint16_t*)c->rest;
  a.lse = c->lse;
  return a;
}

}  // namespace

RESS_API int ress_block_attn_fwd(const ress_block_attn* c, hipStream_t stream) {
  RESS_REQUIRE(c, "ress_block_attn_fwd: null arguments");
  AttnArgs a = arguments(c);
  const int D = c->head_dim, dtype = c->dtype;
  if (int rc = check(a, D, dtype, "ress_block_attn_fwd")) return rc;
  if (!a.B || !a.Hq || !a.Tq) return 0;
  RESS_REQUIRE(fits(a.q, a.Hq, a.Tq, D) && fits(a.o, a.Hq, a.Tq, D) && (a.Tk == 0 || (fits(a.k, a.Hk, a.Tk, D) && fits(a.v, a.Hk, a.Tk, D))),
               "ress_block_attn_fwd: operands must be 16-byte aligned, strides multiples of 8, tokens at least head_dim apart");
  unsigned blocks;
  if (int rc = grid((long long)a.B * a.Hq * cdiv(a.Tq, QB), 256, "ress_block_attn_fwd", &blocks)) return rc;
  RESS_BA_EACH({
    if (a.map) hipLaunchKernelGGL((k_block_attn_fwd<DT, DIM, true>), dim3(blocks), dim3(256), bit_bytes(cdiv(a.Tk, KB)), stream, a);
    else hipLaunchKernelGGL((k_block_attn_fwd<DT, DIM, false>), dim3(blocks), dim3(256), 0, stream, a);
  })
  RESS_LAUNCHED("k_block_attn_fwd");
  return 0;
}

RESS_API long long ress_block_attn_bwd_workspace_size(const ress_block_attn* c) {
  if (!c || c->B < 0 || c->q_heads < 0 || c->kv_heads < 0 || c->Tq < 0) return -1;
  return 8ll * c->B * c->q_heads * c->Tq + 8ll * c->B * c->kv_heads;
}

RESS_API int ress_block_attn_bwd(const ress_block_attn* c, const ress_strided* grad_out, const ress_strided* dq,
                                 const ress_strided* dk, const ress_strided* dv, void* workspace, long long workspace_bytes,
                                 hipStream_t stream) {
  const char* name = "ress_block_attn_bwd";
  RESS_REQUIRE(c && grad_out && dq && dk && dv, "%s: null arguments", name);
  AttnArgs a = arguments(c);
  a.go = view(*grad_out);
  a.dq = view(*dq);
  a.dk = view(*dk);
  a.dv = view(*dv);
  const int D = c->head_dim, dtype = c->dtype;
  if (int rc = check(a, D, dtype, name)) return rc;
  if (!a.B || !a.Hq) return 0;
  RESS_REQUIRE((a.Tq == 0 || (fits(a.q, a.Hq, a.Tq, D) && fits(a.o, a.Hq, a.Tq, D) && fits(a.go, a.Hq, a.Tq, D) && fits(a.dq, a.Hq, a.Tq, D))) &&
                   (a.Tk == 0 || (fits(a.k, a.Hk, a.Tk, D) && fits(a.v, a.Hk, a.Tk, D) && fits(a.dk, a.Hk, a.Tk, D) && fits(a.dv, a.Hk, a.Tk, D))),
               "%s: operands must be 16-byte aligned, strides multiples of 8, tokens at least head_dim apart", name);
  RESS_REQUIRE(a.Tq == 0 || (a.rest && ((uintptr_t)a.rest & 15) == 0 && a.lse), "%s: the forward pass's rest and lse are needed", name);
  RESS_REQUIRE(workspace_bytes >= ress_block_attn_bwd_workspace_size(c) && (workspace || !workspace_bytes), "%s: the workspace is too small", name);
  const long long rows = (long long)a.B * a.Hq * a.Tq;
  a.lse_b = (float*)workspace;
  a.ndelta = a.lse_b + rows;
  a.top = (uint32_t*)(a.ndelta + rows);
  const bool wide = !a.map;  // 128 keys a workgroup; under a map one of its key blocks
  const int keys = wide ? 128 : 64, chunks = cdiv(a.Tk, VTOP_ROWS);
  unsigned qblocks = 0, kblocks = 0, dblocks = 0, vblocks = 0;
  if (int rc = grid((long long)a.B * a.Hq * cdiv(a.Tq, QB), 256, name, &qblocks)) return rc;
  if (int rc = grid((long long)a.B * a.Hk * cdiv(a.Tk, keys), 2 * keys, name, &kblocks)) return rc;
  const int dchunks = cdiv(a.Tq, DELTA_ROWS);
  if (int rc = grid((long long)a.B * a.Hq * dchunks, 256, name, &dblocks)) return rc;
  if (int rc = grid((long long)a.B * a.Hk * chunks, 256, name, &vblocks)) return rc;
  if (dtype == BA_F16 && a.Tk) {
    hipLaunchKernelGGL(k_block_attn_clear, dim3(cdiv(2 * a.B * a.Hk, 256)), dim3(256), 0, stream, a.top, 2 * a.B * a.Hk);
    if (D == 64) hipLaunchKernelGGL((k_block_attn_vtop<64>), dim3((unsigned)((long long)a.B * a.Hk * chunks)), dim3(256), 0, stream, a, chunks);
    else hipLaunchKernelGGL((k_block_attn_vtop<128>), dim3((unsigned)((long long)a.B * a.Hk * chunks)), dim3(256), 0, stream, a, chunks);
    RESS_LAUNCHED("k_block_attn_vtop");
  }
  RESS_BA_EACH({
    if (a.Tq) {
      hipLaunchKernelGGL((k_block_attn_delta<DT, DIM>), dim3((unsigned)((long long)a.B * a.Hq * dchunks)), dim3(256), 0, stream, a, dchunks);
      RESS_LAUNCHED("k_block_attn_delta");
      if (a.map) hipLaunchKernelGGL((k_block_attn_dq<DT, DIM, true>), dim3(qblocks), dim3(256), bit_bytes(cdiv(a.Tk, KB)), stream, a);
      else hipLaunchKernelGGL((k_block_attn_dq<DT, DIM, false>), dim3(qblocks), dim3(256), 0, stream, a);
      RESS_LAUNCHED("k_block_attn_dq");
    }
    if (a.Tk) {
      if (a.map) hipLaunchKernelGGL((k_block_attn_dkv<DT, DIM, 2, true>), dim3(kblocks), dim3(128), bit_bytes(cdiv(a.Tq, QB)), stream, a);
      else hipLaunchKernelGGL((k_block_attn_dkv<DT, DIM, 4, false>), dim3(kblocks), dim3(256), 0, stream, a);
      RESS_LAUNCHED("k_block_attn_dkv");
    }
  })
  return 0;
}
