// The paged 8-bit key/value cache of a streamed sequence: its layout and the device helpers that the
// kernels writing it (kvcache.hip) and the attention reading it (cache_attn.hip) share.
//
// A page holds KV_PAGE = 64 tokens of one key/value head (the framework's key block):
//   k_codes [n_pages][H][64 tokens][D]   8-bit codes of the keys
//   v_codes [n_pages][H][D][64 places]   8-bit codes of the values, transposed; place p holds token
//           v_token(p), so that the 16 bytes a lane of the 16x16x32 MFMA reads as its A operand (V^T)
//           for two products lie together in the order in which P comes out of the scores' product
//   k_scale, v_scale [n_pages][H] f32    value = code * scale
// A sequence's unfinished page is held in 16 bits, by slot: tail_k [slots][H][64][D], tail_v
// [slots][H][D][64 places], and tail_top [slots][H] f32, the largest |value| in tail_v (NaN once one is
// not finite). What a page holds depends on its tokens alone, not on the calls they came in.
#pragma once
#include "../../include/ress_hip.h"
#include "common.h"

constexpr int KV_PAGE = 64;
constexpr int KV_LINE = 32;                // ints from one slot's `arrived` to the next: a cache line
constexpr int KV_I8 = 0, KV_FP8 = 1;       // ress_kv_cache.codes
constexpr int KV_BF16 = 1, KV_F16 = 2;     // ress_kv_cache.dtype
// ress_kv_cache.status bits
constexpr int KV_ST_FULL = 1, KV_ST_POS = 2, KV_ST_PAGE = 4, KV_ST_NONFINITE = 8, KV_ST_SLOT = 16;

// Checks a cache handle on the host (kvcache.hip): 0, or -1 with the message set.
int ress_kv_check(const ress_kv_cache* c, int B, const char* who);

// The slot of a batch's row, and whether it lies in the cache: one that does not (its number on the device was changed, or
// freed under a recorded graph) is reported, and its row is one of no tokens.
__device__ __forceinline__ int slot_of(const ress_kv_cache& c, const int* slots, int b, bool& ok) {
  const int s = slots ? slots[b] : b;
  ok = s >= 0 && s < c.max_seqs;
  return ok ? s : 0;
}

// Tokens of a slot, as the kernels take them: between none and what its pages (or, for a reader, a table) have room for,
// so that lengths changed from outside, as by a snapshot whose recording never ran, reach no memory but the slot's.
__device__ __forceinline__ int held_tokens(int len, int pages) { return min(max(len, 0), pages * KV_PAGE); }

// A launch counts its threads in 32 bits.
inline bool launchable(long long workgroups, long long threads) { return workgroups * threads < (1ll << 32); }

// the token of place p of a value row: p = 16h + 8u + 4g + r  <->  token 32u + 16g + 4h + r
__host__ __device__ constexpr __forceinline__ int v_token(int p) {
  return ((p >> 3) & 1) * 32 + ((p >> 2) & 1) * 16 + (p >> 4) * 4 + (p & 3);
}
__host__ __device__ constexpr __forceinline__ int v_place(int t) {
  return ((t >> 2) & 3) * 16 + (t >> 5) * 8 + ((t >> 4) & 1) * 4 + (t & 3);
}

// 16-bit element types as their bits
template <int DT>
struct Elem;
template <>
struct Elem<KV_BF16> {
  static constexpr uint32_t INF = 0x7f80u;
  static __device__ __forceinline__ float get(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
  static __device__ __forceinline__ uint16_t put(float f) { return (uint16_t)f32_to_bf16_bits(f); }
};
template <>
struct Elem<KV_F16> {
  static constexpr uint32_t INF = 0x7c00u;
  static __device__ __forceinline__ float get(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }
  static __device__ __forceinline__ uint16_t put(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
};

typedef short v2s __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

// Four 8-bit codes as four elements of the 16-bit type, exactly (an int8 or e4m3 value fits both).
template <int DT, int CODES>
__device__ __forceinline__ uint2 widen4(uint32_t w) {
  uint2 r;
  if constexpr (CODES == KV_FP8) {
    if constexpr (DT == KV_BF16) {
      r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
      r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
    } else {
      r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
      r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    }
  } else if constexpr (DT == KV_F16) {
    // 0x6400 | u is 1024 + u for u = code + 128 (0..255), and taking 1152 away is exact
    const uint32_t u = w ^ 0x80808080u;
    const v2h off = {(_Float16)1152.0f, (_Float16)1152.0f};
    const v2h a = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
    const v2h b = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
    r.x = __builtin_bit_cast(uint32_t, a - off);
    r.y = __builtin_bit_cast(uint32_t, b - off);
  } else {
    // an 8-bit integer in fp32 has its bits in the upper half, which is its bf16
    const float f0 = (float)(int)(int8_t)(w & 0xffu), f1 = (float)(int)(int8_t)((w >> 8) & 0xffu);
    const float f2 = (float)(int)(int8_t)((w >> 16) & 0xffu), f3 = (float)(int)(int8_t)(w >> 24);
    r.x = __builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x07060302u);
    r.y = __builtin_amdgcn_perm(__float_as_uint(f3), __float_as_uint(f2), 0x07060302u);
  }
  return r;
}

// The float that one code stands for (before its scale).
template <int CODES>
__device__ __forceinline__ float code_value(uint8_t c) {
  if constexpr (CODES == KV_I8) return (float)(int8_t)c;
  else return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}

template <int CODES>
__host__ __device__ constexpr float code_max() { return CODES == KV_I8 ? 127.0f : 448.0f; }

// Four values (already times the inverse scale) as codes, rounded to nearest, ties to even.
template <int CODES>
__device__ __forceinline__ uint32_t narrow4(float a, float b, float c, float d) {
  constexpr float M = code_max<CODES>();
  a = fminf(fmaxf(a, -M), M);
  b = fminf(fmaxf(b, -M), M);
  c = fminf(fmaxf(c, -M), M);
  d = fminf(fmaxf(d, -M), M);
  if constexpr (CODES == KV_FP8) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  } else {
    const uint32_t x = (uint32_t)(int)rintf(a), y = (uint32_t)(int)rintf(b), z = (uint32_t)(int)rintf(c),
                   w = (uint32_t)(int)rintf(d);
    return (x & 0xffu) | ((y & 0xffu) << 8) | ((z & 0xffu) << 16) | (w << 24);
  }
}

// Eight consecutive 16-bit elements: one access where everything is 16-byte aligned (`vec`), else eight.
__device__ __forceinline__ uint4 ld8(const uint16_t* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint16_t elem8(const uint4& v, int i) {
  const uint32_t w = i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w;
  return (uint16_t)(i & 1 ? w >> 16 : w & 0xffffu);
}
__device__ __forceinline__ uint4 pack8(const uint16_t (&e)[8]) {
  return make_uint4(e[0] | ((uint32_t)e[1] << 16), e[2] | ((uint32_t)e[3] << 16), e[4] | ((uint32_t)e[5] << 16),
                    e[6] | ((uint32_t)e[7] << 16));
}
