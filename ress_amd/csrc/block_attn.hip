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
// P and dS are rounded to the operands' type for that; FINE: what the rounding took is multiplied too (of dQ's half in any case).
// Transposed A operands (V^T, K^T, dO^T, Q^T) come out of the row-major LDS tiles by ds_read_tr16_b64, which gives lane i of 16 the
// i-th column of a 4 x 16 block. dQ and dK/dV are kernels of their own, each the owner of its rows: S and dP are computed
// twice (with dQ's half in two terms 19 products' worth of operations for the 14 that a step needs), and nothing is added by
// atomics, so results repeat bit for bit.
#include "../../include/ress_hip.h"
#include "block_attn.h"

namespace {

constexpr int NS = 3;  // LDS stages
// Below this many tiles of 128 keys (2.5 workgroups a CU) dK and dV's are tiles of 64 keys, twice as many. In us, 128 keys / 64: 16 heads of
// 1,374 in bf16, 176 tiles 31 / 29, 352 43 / 43, 528 65 / 66, 704 72 / 80, 2,816 268 / 300; a head of 128, causal, 2,048 tokens, four query
// heads a key head in fp16, 256 tiles 232 / 217, 512 417 / 332, 640 444 / 415, 768 495 / 485, 1,024 620 / 643.
constexpr int WIDE_TILES = 640;

// ---- forward ----------------------------------------------------------------
// A wave has 32 queries. Steps of 64 keys, at a head of 128 in two stages (three of 32 keys 153 us for 135, the causal case).
// Bound by the vector unit where the card is full: of a step's 16 products (D = 64) and 32 exponentials a lane, the latter are
// four times as dear as other instructions.
template <int DT, int D, bool MAP, bool FINE>
__global__ __launch_bounds__(256, FINE ? 1 : D == 64 ? 3 : 2) void k_block_attn_fwd(AttnArgs a) {
  constexpr int SR = 64, KT = SR / 32, TILE = SR * 2 * D, NS = D == 64 ? 3 : 2;
  __shared__ __align__(16) uint8_t lds[NS][2 * TILE];
  extern __shared__ uint32_t bits[];
  const unsigned lds0 = lds_address(lds);
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
    const int whole = (a.causal ? min(hd.klen, max(0, q0 + off + 1)) : hd.klen) / SR;  // steps that every row sees whole
    uint4 q[D / 16];
    load_row<D>(a.q, it.b, it.h, row, row < qlen, ln.half, q);
    const int steps = cdiv(most, SR);
    const Walk<MAP, KB / SR> walk(a.map + it.b * a.mb + it.h * a.mh + it.tile * a.mq, a.mk, part_of(steps, blockIdx.y, a.parts),
                                  part_of(steps, blockIdx.y + 1, a.parts), bits, false);
    const Stream<D, 4, SR> ks(a.k, hd.kbase(a.k), ln), vs(a.v, hd.kbase(a.v), ln);
    auto fetch = [&](int stage, int st) {
      ks.fetch(lds0 + stage * 2 * TILE, st * SR, hd.klen, w);
      vs.fetch(lds0 + stage * 2 * TILE + TILE, st * SR, hd.klen, w);
    };
    auto compute = [&](auto mask_tag, const uint8_t* tile, int st) {
      v16f s[KT];
      each<KT>([&](auto t) { s[t] = rows_times<DT, D>(tile, 32 * t, ln, q, zero16()); });
      if constexpr (decltype(mask_tag)::value) {
        const int below = sees - st * SR - 4 * ln.half;
        each<KT>([&](auto t) {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[t][r] = 32 * t + c_row(r) < below ? s[t][r] : -__builtin_huge_valf();
        });
      }
      // Whether a score lies more than LAZY above m. Where m + LAZY is not negative only positive scores can, and they
      // order as their bits do: integer maxima of three, which need no quieting of NaNs.
      int top = 0;
      each<KT>([&](auto t) {
#pragma unroll
        for (int r = 0; r < 16; ++r) top = max(top, __float_as_int(s[t][r]));
      });
      if (__any(__int_as_float(top) * a.scale2 > m + LAZY || m + LAZY < 0.0f)) {
        float x = LOWEST;
        each<KT>([&](auto t) {
#pragma unroll
          for (int r = 0; r < 16; ++r) x = fmaxf(x, s[t][r]);
        });
        x = pair_max(x);
        x = x == LOWEST ? LOWEST : x * a.scale2;
        const float mn = x > m + LAZY ? x : m;  // a row moves by its own scores, so its bits do not hang on its neighbours
        const float f = exp2f(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= f;
      }
      each<KT>([&](auto t) {
        float e[16];
        uint4 p[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(s[t][r], a.scale2, -m));
        pack16<DT>(e, p);
        // the sum before P is rounded: the backward pass forms P from it
        l += sum16(e);
        each<D / 32>([&](auto d) { o[d] = columns_times<DT, D>(tile + TILE, 32 * t, d, ln, p, o[d]); });
        if constexpr (FINE) {
          uint4 rest[2];
          pack_rest<DT>(e, p, rest);
          each<D / 32>([&](auto d) { o[d] = columns_times<DT, D>(tile + TILE, 32 * t, d, ln, rest, o[d]); });
        }
      });
    };
    run_steps<NS, 2 * ks.DMAS>(
        walk, fetch, [&](int st) { return st < whole; },
        [&](int stage, int st) { compute(std::false_type{}, lds[stage], st); },
        [&](int stage, int st) { compute(std::true_type{}, lds[stage], st); });
  }
  l = pair_sum(l);
  const bool some = row < qlen && (l > 0.0f || l != l);
  if (row >= a.Tq) return;
  if (a.parts > 1) {
    const long long r = (long long)blockIdx.y * a.B * a.Hq * a.Tq + a.row_at(it, row);
    store_part<D>(a.part + r * D, ln.half, o, 1.0f / l, some);
    if (ln.half == 0) a.part2[r] = some ? m + log2f(l) : -__builtin_huge_valf();
  } else {
    store_out<DT, D>(a, it, row, ln.half, o, 1.0f / l, some);
    if (a.lse && ln.half == 0) a.lse[a.row_at(it, row)] = some ? m + log2f(l) : __builtin_huge_valf();
  }
}

// ---- backward: row sums -----------------------------------------------------
// -delta_i = -dO_i.(o_i + what o's rounding took), and lse less the lift of P. Bound by its bytes: 21,904 rows of 16 heads 24 us,
// 5.7 TB/s.
template <int DT, int D>
__global__ __launch_bounds__(256) void k_block_attn_delta(AttnArgs a, int chunks) {
  constexpr int LR = D / 8;
  const int bh = blockIdx.x / chunks, b = bh / a.Hq, h = bh % a.Hq, piece = threadIdx.x % LR;
  const int from = blockIdx.x % chunks * DELTA_ROWS, end = min(a.Tq, from + DELTA_ROWS), qlen = a.q_len(b);
  for (int i = from + threadIdx.x / LR; i < end; i += 256 / LR) {  // a row's lanes go together
    float sum = 0.0f;
    const long long r = (long long)bh * a.Tq + i;
    if (i < qlen) {
      float x[8], y[8], z[8];
      unpack8<DT>(*reinterpret_cast<const uint4*>(a.go.at(b, h, i) + 8 * piece), x);
      unpack8<DT>(*reinterpret_cast<const uint4*>(a.o.at(b, h, i) + 8 * piece), y);
      unpack8<DT>(*reinterpret_cast<const uint4*>(a.rest + r * D + 8 * piece), z);
#pragma unroll
      for (int u = 0; u < 8; ++u) sum = fmaf(x[u], y[u] + z[u], sum);
    }
#pragma unroll
    for (int s = 1; s < LR; s <<= 1) sum += __shfl_xor(sum, s, LR);
    if (piece == 0) {
      a.ndelta[r] = -sum;
      a.lse_b[r] = a.lse[r] - lift(DT);
    }
  }
}

// fp16: dS is formed times a power of two, one for each row of dQ and each key of dK, so that a gradient far below fp16's smallest
// number keeps its bits and nothing takes them but what the row or the key itself meets: 2^60 to begin with (fp32 holds that
// times the largest dP - delta there is, 2^41), and where a |dS| passes 2^15, less by what takes that below 2^12, with the sum so far.
constexpr float DS_LIFT = 60.0f;
// Whether a row (key) of the wave has such a one; high: the lane's largest
__device__ __forceinline__ bool over(const float (&e)[16], float lift, float& high) {
  high = 0.0f;
#pragma unroll
  for (int r = 0; r < 16; ++r) high = fmaxf(high, fabsf(e[r]));
  high *= lift;
  return __any(high > 0x1p15f);
}
__device__ __forceinline__ int shift_of(float high) {
  high = pair_max(high);  // the row's (key's) other half decides alike; what is not finite makes the row so whatever the shift is
  return high > 0x1p15f && high < __builtin_huge_valf() ? 12 - __builtin_amdgcn_frexp_expf(high) : 0;
}
template <int N>
__device__ __forceinline__ void scale_all(v16f (&acc)[N], float by) {
#pragma unroll
  for (int d = 0; d < N; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] *= by;
}

// ---- backward: dQ -----------------------------------------------------------
// A wave has 32 queries and their gradients as operands. Bound by matrix and vector unit in turn (16 frames of 1,374 tokens, 30% of the
// blocks: products 53% of the cycles, vector instructions 62%), at a clock that their power brings down to some 1.7 GHz.
template <int DT, int D, bool MAP, bool FINE>
__global__ __launch_bounds__(256, FINE ? 1 : D == 64 ? 3 : 2) void k_block_attn_dq(AttnArgs a) {
  constexpr int SR = step_rows(D), KT = SR / 32, TILE = SR * 2 * D;
  __shared__ __align__(16) uint8_t lds[NS][2 * TILE];
  extern __shared__ uint32_t bits[];
  const unsigned lds0 = lds_address(lds);
  const Lane<D> here;
  Item it;
  if (!it.query_tile(a)) return;
  const Head hd(a, it.b, it.h / a.G);
  const int qlen = a.q_len(it.b), q0 = it.tile * QB;
  const int w = here.wave, row = q0 + 32 * w + here.c32;
  v16f dq[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d) dq[d] = zero16();
  float up = DT == BA_F16 ? exp2f(DS_LIFT) : 1.0f;  // dS's lift
  if (q0 < qlen) {
    const int off = hd.klen - qlen;
    const int sees = a.causal ? min(hd.klen, max(0, row + off + 1)) : hd.klen;
    const int last = min(q0 + QB, qlen) - 1;
    const int most = a.causal ? min(hd.klen, max(0, last + off + 1)) : hd.klen;
    const int whole = (a.causal ? min(hd.klen, max(0, q0 + off + 1)) : hd.klen) / SR;
    uint4 q[D / 16], g[D / 16];
    load_row<D>(a.q, it.b, it.h, row, row < qlen, here.half, q);
    load_row<D>(a.go, it.b, it.h, row, row < qlen, here.half, g);
    float lse = 0.0f, nd = 0.0f;
    if (row < qlen) {
      lse = a.lse_b[a.row_at(it, row)] + lift(DT) - (DT == BA_F16 ? DS_LIFT : 0.0f);
      nd = a.ndelta[a.row_at(it, row)];
    }
    // -delta is added by the matrix cores where 16 registers are to be had for it (2 x 16 products less a step: 144 us for 152 at a
    // head of 128; at 64 they are not, 1,180 for 940)
    v16f ndelta;
#pragma unroll
    for (int r = 0; r < 16; ++r) ndelta[r] = nd;
    const int steps = cdiv(most, SR);
    const Walk<MAP, KB / SR> walk(a.map + it.b * a.mb + it.h * a.mh + it.tile * a.mq, a.mk, part_of(steps, blockIdx.y, a.parts),
                                  part_of(steps, blockIdx.y + 1, a.parts), bits, false);
    const Stream<D, 4, SR> ks(a.k, hd.kbase(a.k), here), vs(a.v, hd.kbase(a.v), here);
    auto fetch = [&](int stage, int st) {
      ks.fetch(lds0 + stage * 2 * TILE, st * SR, hd.klen, w);
      vs.fetch(lds0 + stage * 2 * TILE + TILE, st * SR, hd.klen, w);
    };
    auto compute = [&](auto mask_tag, const uint8_t* tile, int st) {
      const Lane<D> ln = here.anew();
      each<KT>([&](auto t) {
        const v16f s = rows_times<DT, D>(tile, 32 * t, ln, q, zero16());
        const v16f dp = rows_times<DT, D>(tile + TILE, 32 * t, ln, g, D == 128 ? ndelta : zero16());
        float e[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, -lse)) * (D == 128 ? dp[r] : dp[r] + nd);
        if constexpr (decltype(mask_tag)::value) {
          const int below = sees - st * SR - 4 * ln.half;
#pragma unroll
          for (int r = 0; r < 16; ++r) e[r] = 32 * t + c_row(r) < below ? e[r] : 0.0f;
        }
        if constexpr (DT == BA_F16) {
          float high;
          if (over(e, 1.0f, high)) {
            const int shift = shift_of(high);
            const float by = ldexpf(1.0f, shift);
#pragma unroll
            for (int r = 0; r < 16; ++r) e[r] *= by;
            scale_all(dq, by);
            lse -= shift;
            up *= by;
          }
        }
        uint4 ds[2];
        pack16<DT>(e, ds);
        each<D / 32>([&](auto d) { dq[d] = columns_times<DT, D>(tile, 32 * t, d, ln, ds, dq[d]); });
        // Half of dS, or all (FINE), in two terms: its rows add up to 0, and what its rounding and delta's (P's in the forward pass) make of
        // that sum goes into dQ times what the keys have in common. Keys with an offset of half their deviation, bf16: dQ off by 2.7e-3 in
        // one term, 2.4e-3 so (1.7e-3 is the result's rounding); four frames 72 us for 60. Taking the sum out times some mean of the keys
        // is cheaper, but lets keys in that the row does not see or that weigh nothing for it.
        auto fine = [&] {
          uint4 rest[2];
          pack_rest<DT>(e, ds, rest);
          each<D / 32>([&](auto d) { dq[d] = columns_times<DT, D>(tile, 32 * t, d, ln, rest, dq[d]); });
        };
        if constexpr (FINE || (KT == 2 && decltype(t)::value == 0)) fine();
        else if constexpr (KT == 1) {
          if (!(st & 1)) fine();
        }
      });
    };
    run_steps<NS, 2 * ks.DMAS>(
        walk, fetch, [&](int st) { return st < whole; },
        [&](int stage, int st) { compute(std::false_type{}, lds[stage], st); },
        [&](int stage, int st) { compute(std::true_type{}, lds[stage], st); });
  }
  if (row >= a.Tq) return;
  if (a.parts > 1)
    store_part<D>(a.part + ((long long)blockIdx.y * a.B * a.Hq * a.Tq + a.row_at(it, row)) * D, here.half, dq, a.scale / up, row < qlen);
  else
    store_grad<DT, D>(a.dq, it.b, it.h, row, here.half, dq, a.scale / up, row < qlen);
}

// ---- backward: dK and dV ----------------------------------------------------
// A wave has 32 keys; queries and their gradients stream past. At a head of 64 bound by the products and what stands between them (16
// sparse frames: matrix cores 47% of the cycles, vector unit 43%, waves waiting 44%). At a head of 128 no register is left to read
// LDS far ahead, and a wave alone on its SIMD takes 1.5 us a step of 32 queries of which the products are 0.6; two share it at 2.1
// (full card: matrix cores 47%). Tried there: 64 keys a wave, one wave a SIMD, every operand read meeting two tiles, no wave waiting
// for another: 502 us for 281. The tiles of a causal launch cut in two by their steps: 250 us and 40 to join them for 244.
// Four waves of 32 keys, or SPLIT (under a map, where a workgroup has one key block, and where tiles are few): two waves of 32
// keys take the first 32 queries of each step, two more with the same keys the others, and their sums are added at the end.
template <int DT, int D, bool SPLIT, bool MAP, bool FINE>
__global__ __launch_bounds__(256, FINE ? 1 : D == 64 ? 3 : 2) void k_block_attn_dkv(AttnArgs a) {
  constexpr int SR = SPLIT ? 64 : step_rows(D), KT = SR / 32, TILE = SR * 2 * D, STAGE = 2 * TILE + 512;
  constexpr int KEYS = SPLIT ? 64 : 128, STAGES = SPLIT && D == 128 ? 2 : NS;
  __shared__ __align__(16) uint8_t lds[STAGES][STAGE];
  extern __shared__ uint32_t bits[];
  const unsigned lds0 = lds_address(lds);
  const Lane<D> here;
  Item it;
  if (!it.key_tile(a, KEYS)) return;
  const Head hd(a, it.b, it.h);
  const int qlen = a.q_len(it.b), k0 = it.tile * KEYS;
  const int w = here.wave, key = k0 + 32 * (SPLIT ? w & 1 : w) + here.c32;
  v16f dk[D / 32], dv[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d) dk[d] = dv[d] = zero16();
  float fp = DT == BA_F16 ? exp2f(DS_LIFT - lift(DT)) : 1.0f;  // P's lift to dS's
  if (k0 < hd.klen && qlen > 0) {
    const int off = hd.klen - qlen;
    uint4 k[D / 16], v[D / 16];
    load_row<D>(a.k, it.b, it.h, key, key < hd.klen, here.half, k);
    load_row<D>(a.v, it.b, it.h, key, key < hd.klen, here.half, v);
    const int from = a.causal ? min(qlen, max(0, k0 - off)) : 0;      // no row before it sees a key of the tile
    const int whole = a.causal ? max(0, k0 + KEYS - 1 - off) : 0;     // rows from here on see all of it
    const int first = a.causal ? key - off - 4 * here.half : 0;         // rows from `first` on see the lane's key
    // the steps of all heads that share the keys, one after the other, cut into parts
    const int steps = cdiv(qlen, SR), lo = part_of(steps * a.G, blockIdx.y, a.parts), hi = part_of(steps * a.G, blockIdx.y + 1, a.parts);
    for (int g = lo / steps; g * steps < hi; ++g) {
      const int h = it.h * a.G + g;
      const Walk<MAP, QB / SR> walk(a.map + it.b * a.mb + h * a.mh + k0 / KB * a.mk, a.mq, max(from / SR, lo - g * steps),
                                    min(steps, hi - g * steps), bits, g * steps > lo);
      const Stream<D, 4, SR> qs(a.q, a.q.at(it.b, h, 0), here), gs(a.go, a.go.at(it.b, h, 0), here);
      const float* values = ((w & 1) ? a.ndelta : a.lse_b) + ((long long)it.b * a.Hq + h) * a.Tq;
      auto fetch = [&](int stage, int st) {
        const unsigned to = lds0 + stage * STAGE;
        qs.fetch(to, st * SR, qlen, w);
        gs.fetch(to + TILE, st * SR, qlen, w);
        // the rows' values, by every wave, so that all have as many DMAs in flight
        fetch_row_values(values + st * SR, min(SR, qlen - st * SR), to + 2 * TILE + 256 * (w & 1));
      };
      auto compute = [&](auto mask_tag, const uint8_t* tile, int st) {
        const Lane<D> ln = here.anew();
        each<SPLIT ? 1 : KT>([&](auto t_) {
          const int t = SPLIT ? w >> 1 : (int)t_;
          const v16f s = rows_times<DT, D>(tile, 32 * t, ln, k, zero16());
          float e[16];
          {
            const v16f lse = row_values(tile + 2 * TILE, 32 * t, ln);
#pragma unroll
            for (int r = 0; r < 16; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, -lse[r]));
          }
          if constexpr (decltype(mask_tag)::value) {
#pragma unroll
            for (int r = 0; r < 16; ++r) e[r] = st * SR + 32 * t + c_row(r) >= first ? e[r] : 0.0f;
          }
          uint4 p[2], ds[2], rest[2];
          pack16<DT>(e, p);
          if constexpr (FINE) pack_rest<DT>(e, p, rest);
          if constexpr (D == 128) __builtin_amdgcn_sched_barrier(0);  // reads ahead of their use would take registers that are not there
          const v16f dp = rows_times<DT, D>(tile + TILE, 32 * t, ln, v, row_values(tile + 2 * TILE + 256, 32 * t, ln));
          each<D / 32>([&](auto x) { dv[x] = columns_times<DT, D>(tile + TILE, 32 * t, x, ln, p, dv[x]); });
          if constexpr (FINE) each<D / 32>([&](auto x) { dv[x] = columns_times<DT, D>(tile + TILE, 32 * t, x, ln, rest, dv[x]); });
          if constexpr (DT == BA_F16) {
            // products of their own: with dS itself formed in front of the branch its registers are not to be had (dK and dV 290 us for 246)
            float ds[16], high;
#pragma unroll
            for (int r = 0; r < 16; ++r) ds[r] = e[r] * dp[r];
            if (over(ds, fp, high)) {
              const float by = ldexpf(1.0f, shift_of(high));
              scale_all(dk, by);
              fp *= by;
            }
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            if constexpr (DT == BA_F16) e[r] *= fp;
            e[r] *= dp[r];
          }
          pack16<DT>(e, ds);
          each<D / 32>([&](auto x) { dk[x] = columns_times<DT, D>(tile, 32 * t, x, ln, ds, dk[x]); });
          if constexpr (FINE) {
            pack_rest<DT>(e, ds, rest);
            each<D / 32>([&](auto x) { dk[x] = columns_times<DT, D>(tile, 32 * t, x, ln, rest, dk[x]); });
          }
        });
      };
      run_steps<STAGES, 2 * qs.DMAS + 1>(
          walk, fetch, [&](int st) { return st * SR < whole; },
          [&](int stage, int st) { compute(std::true_type{}, lds[stage], st); },
          [&](int stage, int st) { compute(std::false_type{}, lds[stage], st); });
    }
  }
  float by_k = a.scale;
  const float by_v = DT == BA_F16 ? 0x1p-14f : 1.0f;
  if constexpr (DT == BA_F16) by_k = a.scale * 0x1p-14f / fp;
  if constexpr (SPLIT) {
    if constexpr (DT == BA_F16) {  // the two waves' lifts differ
      scale_all(dk, by_k);
      by_k = 1.0f;
    }
    // waves 2 and 3 hand their sums to 0 and 1, dK's and then dV's: 16 floats of a lane and tile of 32 dims
    static_assert(2 * (D / 32) * 16 * 64 * 4 <= (int)sizeof(lds), "the sums fit the stages");
    float* to = reinterpret_cast<float*>(&lds[0][0]) + (w & 1) * (D / 32) * 16 * 64 + (threadIdx.x & 63);
    auto add = [&](v16f (&acc)[D / 32]) {
      __syncthreads();
      if (w >= 2) each<D / 32>([&](auto x) {
#pragma unroll
        for (int r = 0; r < 16; ++r) to[(x * 16 + r) * 64] = acc[x][r];
      });
      __syncthreads();
      if (w < 2) each<D / 32>([&](auto x) {
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[x][r] += to[(x * 16 + r) * 64];
      });
    };
    add(dk);
    add(dv);
    if (w >= 2) return;
  }
  if (key >= a.Tk) return;
  if (a.parts > 1) {
    const long long r = (((long long)blockIdx.y * a.B + it.b) * a.Hk + it.h) * a.Tk + key;
    store_part<D>(a.part + r * D, here.half, dk, by_k, key < hd.klen);
    store_part<D>(a.part2 + r * D, here.half, dv, by_v, key < hd.klen);
  } else {
    store_grad<DT, D>(a.dk, it.b, it.h, key, here.half, dk, by_k, key < hd.klen);
    store_grad<DT, D>(a.dv, it.b, it.h, key, here.half, dv, by_v, key < hd.klen);
  }
}

// ---- parts joined -----------------------------------------------------------
// A row a wave: D / 4 lanes take four dims each, and the wave's 256 / D groups of them every 256 / D-th part. OUT:
// o = sum of 2^(lse_p - L) o_p over sum of 2^(lse_p - L), L the largest; else the sum of the parts.
template <int DT, int D, bool OUT>
__global__ __launch_bounds__(256) void k_block_attn_join(AttnArgs a, const float* __restrict__ part, const float* __restrict__ lse, View to,
                                                         int heads, int T) {
  constexpr int LR = D / 4, GROUPS = 64 / LR;
  const long long rows = (long long)a.B * heads * T, r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  const int lane = threadIdx.x & 63, group = lane / LR, d = lane % LR * 4;
  const int t = (int)(r % T), bh = (int)(r / T), b = bh / heads, h = bh % heads;
  float top = -__builtin_huge_valf(), sum = 0.0f, mine = top;
  if constexpr (OUT) {  // at most 64 parts
    mine = lane < a.parts ? lse[lane * rows + r] : top;
    top = mine;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const float x = __shfl_xor(top, s, 64);
      top = x > top || x != x ? x : top;
    }
  }
  const bool some = !OUT || top != -__builtin_huge_valf();
  v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int p0 = 0; p0 < a.parts; p0 += GROUPS) {  // every lane goes all the way: lanes ask others for their lse
    const int p = min(p0 + group, a.parts - 1);
    const bool there = p0 + group < a.parts;
    v4f y = *reinterpret_cast<const v4f*>(part + (p * rows + r) * D + d);
    if constexpr (OUT) {
      const float l = __shfl(mine, p, 64), w = there && some && l != -__builtin_huge_valf() ? exp2f(l - top) : 0.0f;
      sum += w;
      y *= w;  // a part that saw nothing is zero
      x += y;
    } else if (there) {
      x += y;
    }
  }
#pragma unroll
  for (int s = LR; s < 64; s <<= 1) {
    sum += __shfl_xor(sum, s, 64);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] += __shfl_xor(x[i], s, 64);
  }
  if (group) return;
  if (OUT && some) x /= sum;
  const uint2 y = make_uint2(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]));
  *reinterpret_cast<uint2*>(to.at(b, h, t) + d) = y;
  if constexpr (OUT) {
    if (a.rest)
      *reinterpret_cast<uint2*>(a.rest + r * D + d) =
          make_uint2(pack2<DT>(x[0] - unpack1<DT>(y.x, 0), x[1] - unpack1<DT>(y.x, 1)),
                     pack2<DT>(x[2] - unpack1<DT>(y.y, 0), x[3] - unpack1<DT>(y.y, 1)));
    if (a.lse && d == 0) a.lse[r] = some ? top + log2f(sum) : __builtin_huge_valf();
  }
}

// ---- host -------------------------------------------------------------------
bool fits(const View& x, int D) {
  return x.p && ((uintptr_t)x.p & 15) == 0 && x.b >= 0 && x.h >= 0 && ((x.b | x.h | x.t) & 7) == 0 && x.t >= D && x.t < 1ll << 24;
}
int check(const AttnArgs& a, int D, int dtype, const char* name) {
  RESS_REQUIRE(D == 64 || D == 128, "%s: head_dim %d (64 or 128)", name, D);
  RESS_REQUIRE(dtype == BA_BF16 || dtype == BA_F16, "%s: dtype code %d", name, dtype);
  RESS_REQUIRE(a.B >= 0 && a.Hq >= 0 && a.Hk >= 1 && a.Tq >= 0 && a.Tk >= 0 && a.Hq % a.Hk == 0, "%s: bad geometry", name);
  RESS_REQUIRE(a.Tq <= 1 << 26 && a.Tk <= 1 << 26, "%s: more than 2^26 tokens", name);
  RESS_REQUIRE((long long)a.Hq / a.Hk * cdiv(a.Tq, 32) < 1ll << 30, "%s: too many query heads of a key/value head", name);
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
// of joined rows: tiles that are cut are few, 384 of 128 rows
unsigned join_blocks(long long rows) { return (unsigned)((rows + 3) / 4); }
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

// Parts that a launch of `tiles` workgroups is cut into, each of at least LEAST steps of 64 rows: as many as fill the card's 512 places
// for workgroups (two a CU) where a quarter of them or more would stay empty. 16 tiles of 80 queries over 21,984 keys: forward 377 us
// whole, 26 in 32 parts and 5 to join them; dQ 330, 27 and 5 (in one term; now 32).
constexpr int PLACES = 512, LEAST = 8, MOST_PARTS = 64;
int parts_of(long long tiles, long long steps) {
  if (tiles <= 0 || tiles > PLACES * 3 / 4) return 1;
  long long n = (PLACES + tiles - 1) / tiles;
  if (n > steps / LEAST) n = steps / LEAST;
  return (int)(n < 1 ? 1 : n > MOST_PARTS ? MOST_PARTS : n);
}
// Calls of up to so many probabilities multiply P and dS in two terms: 1.7e-3 off in bf16 (the result's own rounding) for up to 2.4e-3,
// however many terms stand behind a result. A trade of time for accuracy where a call is small, and the rule goes by the whole call because
// that bounds the time: 16 heads of 126 tokens 29.4 us of kernels, of 128 x 129 in one term 29.4; four of 256 35.3 for 39.4; 64 of 64 22.4
// for 21.5; one of 512 50.5 for 45.4; 1,024 heads of a row over 256 keys 107 for 93; one row over 2^18 keys 351 for 266.
constexpr int FEW = 1 << 18;
// How a call is cut: keys a workgroup of dK and dV has, and the parts of each kernel
struct Plan {
  bool split, fine;
  int q_parts, k_parts;
  long long q_rows, k_rows;
  explicit Plan(const ress_block_attn* c) {
    const long long wide = (long long)c->B * c->kv_heads * cdiv(c->Tk, 128);
    q_rows = (long long)c->B * c->q_heads * c->Tq;
    fine = q_rows <= FEW && q_rows * c->Tk <= FEW;
    split = c->map || fine || wide < WIDE_TILES;
    k_rows = (long long)c->B * c->kv_heads * c->Tk;
    q_parts = parts_of((long long)c->B * c->q_heads * cdiv(c->Tq, QB), cdiv(c->Tk, KB));
    k_parts = parts_of((long long)c->B * c->kv_heads * cdiv(c->Tk, split ? 64 : 128),
                       (long long)cdiv(c->Tq, 64) * (c->q_heads / c->kv_heads));
  }
  long long fwd_bytes(int D) const { return q_parts > 1 ? 4 * q_parts * q_rows * (D + 1) : 0; }
  long long bwd_part_bytes(int D) const {
    const long long q = q_parts > 1 ? 4 * q_parts * q_rows * D : 0, k = k_parts > 1 ? 8 * k_parts * k_rows * D : 0;
    return q > k ? q : k;
  }
};
template <class F>
void with_plan(bool map, bool fine, F f) {
  if (map && fine) f(std::true_type{}, std::true_type{});
  else if (map) f(std::true_type{}, std::false_type{});
  else if (fine) f(std::false_type{}, std::true_type{});
  else f(std::false_type{}, std::false_type{});
}
bool sizes_ok(const ress_block_attn* c) {
  return c && c->B >= 0 && c->q_heads >= 0 && c->kv_heads >= 1 && c->q_heads % c->kv_heads == 0 && c->Tq >= 0 && c->Tk >= 0 &&
         c->Tq <= 1 << 26 && c->Tk <= 1 << 26 && (c->head_dim == 64 || c->head_dim == 128);
}

}  // namespace

RESS_API long long ress_block_attn_fwd_workspace_size(const ress_block_attn* c) {
  return sizes_ok(c) ? Plan(c).fwd_bytes(c->head_dim) : -1;
}

RESS_API int ress_block_attn_fwd(const ress_block_attn* c, void* workspace, long long workspace_bytes, hipStream_t stream) {
  const char* name = "ress_block_attn_fwd";
  RESS_REQUIRE(c, "%s: null arguments", name);
  AttnArgs a = arguments(c);
  const int D = c->head_dim, dtype = c->dtype;
  if (int rc = check(a, D, dtype, name)) return rc;
  if (!a.B || !a.Hq || !a.Tq) return 0;
  RESS_REQUIRE(fits(a.q, D) && fits(a.o, D) && (a.Tk == 0 || (fits(a.k, D) && fits(a.v, D))),
               "%s: operands must be 16-byte aligned, strides multiples of 8, tokens at least head_dim and fewer than 2^24 apart", name);
  const Plan plan(c);
  RESS_REQUIRE(workspace_bytes >= plan.fwd_bytes(D) && ((uintptr_t)workspace & 15) == 0 && (workspace || !plan.fwd_bytes(D)),
               "%s: the workspace is too small or not aligned", name);
  a.parts = plan.q_parts;
  a.part = (float*)workspace;
  a.part2 = a.part + a.parts * plan.q_rows * D;
  unsigned blocks;
  if (int rc = grid((long long)a.B * a.Hq * cdiv(a.Tq, QB), 256 * a.parts, name, &blocks)) return rc;
  RESS_BA_EACH({
    with_plan(a.map, plan.fine, [&](auto map, auto fine) {
      hipLaunchKernelGGL((k_block_attn_fwd<DT, DIM, decltype(map)::value, decltype(fine)::value>), dim3(blocks, a.parts), dim3(256),
                         map ? bit_bytes(cdiv(a.Tk, KB)) : 0, stream, a);
    });
    RESS_LAUNCHED("k_block_attn_fwd");
    if (a.parts > 1) {
      hipLaunchKernelGGL((k_block_attn_join<DT, DIM, true>), dim3(join_blocks(plan.q_rows)), dim3(256), 0, stream, a, a.part, a.part2,
                         a.o, a.Hq, a.Tq);
      RESS_LAUNCHED("k_block_attn_join");
    }
  })
  return 0;
}

RESS_API long long ress_block_attn_bwd_workspace_size(const ress_block_attn* c) {
  if (!sizes_ok(c)) return -1;
  const Plan p(c);
  // 8 bytes a key/value head more than is used: the size stays what it was for callers that have set it aside
  return p.bwd_part_bytes(c->head_dim) + 8 * p.q_rows + 8ll * c->B * c->kv_heads;
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
  if (!a.B) return 0;
  const bool rows = a.Hq && a.Tq;  // without any, dk and dv are zero
  RESS_REQUIRE((!rows || (fits(a.q, D) && fits(a.o, D) && fits(a.go, D) && fits(a.dq, D))) &&
                   (a.Tk == 0 || (fits(a.k, D) && fits(a.v, D) && fits(a.dk, D) && fits(a.dv, D))),
               "%s: operands must be 16-byte aligned, strides multiples of 8, tokens at least head_dim and fewer than 2^24 apart", name);
  RESS_REQUIRE(!rows || (a.rest && ((uintptr_t)a.rest & 15) == 0 && a.lse), "%s: the forward pass's rest and lse are needed", name);
  RESS_REQUIRE(workspace_bytes >= ress_block_attn_bwd_workspace_size(c) && ((uintptr_t)workspace & 15) == 0 && (workspace || !workspace_bytes),
               "%s: the workspace is too small or not aligned", name);
  const Plan plan(c);
  float* const parts = (float*)workspace;  // of dQ and, once these are joined, of dK and dV
  a.lse_b = parts + plan.bwd_part_bytes(D) / 4;
  a.ndelta = a.lse_b + plan.q_rows;
  const int keys = plan.split ? 64 : 128, dchunks = cdiv(a.Tq, DELTA_ROWS);
  unsigned qblocks, kblocks, dblocks;
  if (int rc = grid((long long)a.B * a.Hq * cdiv(a.Tq, QB), 256 * plan.q_parts, name, &qblocks)) return rc;
  if (int rc = grid((long long)a.B * a.Hk * cdiv(a.Tk, keys), 256 * plan.k_parts, name, &kblocks)) return rc;
  if (int rc = grid((long long)a.B * a.Hq * dchunks, 256, name, &dblocks)) return rc;
  RESS_BA_EACH({
    if (rows) {
      hipLaunchKernelGGL((k_block_attn_delta<DT, DIM>), dim3((unsigned)((long long)a.B * a.Hq * dchunks)), dim3(256), 0, stream, a, dchunks);
      RESS_LAUNCHED("k_block_attn_delta");
      a.parts = plan.q_parts;
      a.part = parts;
      with_plan(a.map, plan.fine, [&](auto map, auto fine) {
        hipLaunchKernelGGL((k_block_attn_dq<DT, DIM, decltype(map)::value, decltype(fine)::value>), dim3(qblocks, a.parts), dim3(256),
                           map ? bit_bytes(cdiv(a.Tk, KB)) : 0, stream, a);
      });
      RESS_LAUNCHED("k_block_attn_dq");
      if (a.parts > 1) {
        hipLaunchKernelGGL((k_block_attn_join<DT, DIM, false>), dim3(join_blocks(plan.q_rows)), dim3(256), 0, stream, a, a.part,
                           nullptr, a.dq, a.Hq, a.Tq);
        RESS_LAUNCHED("k_block_attn_join");
      }
    }
    if (a.Tk) {
      a.parts = plan.k_parts;
      a.part = parts;
      a.part2 = parts + a.parts * plan.k_rows * D;
      if (plan.split)
        with_plan(a.map, plan.fine, [&](auto map, auto fine) {
          hipLaunchKernelGGL((k_block_attn_dkv<DT, DIM, true, decltype(map)::value, decltype(fine)::value>), dim3(kblocks, a.parts),
                             dim3(256), map ? bit_bytes(cdiv(a.Tq, QB)) : 0, stream, a);
        });
      else hipLaunchKernelGGL((k_block_attn_dkv<DT, DIM, false, false, false>), dim3(kblocks, a.parts), dim3(256), 0, stream, a);
      RESS_LAUNCHED("k_block_attn_dkv");
      if (a.parts > 1) {
        hipLaunchKernelGGL((k_block_attn_join<DT, DIM, false>), dim3(join_blocks(plan.k_rows)), dim3(256), 0, stream, a, a.part,
                           nullptr, a.dk, a.Hk, a.Tk);
        hipLaunchKernelGGL((k_block_attn_join<DT, DIM, false>), dim3(join_blocks(plan.k_rows)), dim3(256), 0, stream, a, a.part2,
                           nullptr, a.dv, a.Hk, a.Tk);
        RESS_LAUNCHED("k_block_attn_join");
      }
    }
  })
  return 0;
}
