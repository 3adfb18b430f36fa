// The paged KV cache in 8 bits: the object, the two code formats, and what the kernels that write and read it share.
//
// K and V of a (position, kv head) are rows of hd codes with a scale each, value = code * scale:
//   int8   scale = max|x| / 127 rounded up to 4 significant bits (to a multiple of 2^-24 below 2^-21), code = rint(x / scale)
//   e4m3   scale = the least 2^e with max|x| / 2^e <= 448, e >= -15,                                  code = e4m3(x / scale)
// A code has at most 7 significant bits (int8) or 4 (e4m3), so code * scale has at most 11 and is an fp16 number: what
// attends to the cache multiplies fp16 values, exact, and needs no scale inside a sum.  Rounding int8's scale up costs up to an
// eighth of a step (0.5 dB), which is the price of that.  A quotient that is not on a border between two scales is at least
// 2^-12 of itself away from it, since max|x| has 11 significant bits: 32 bits are enough to be exact.
// A value beyond 65504 (rounded up from just below) becomes the next lower code.
// A row with a NaN or an infinity in its K or V has no codes that could stand for it: its K scale is NaN and the V row zero.
// Scores against it are NaN, so every query that sees the position becomes NaN, and no other: a masked NaN is replaced, but a
// masked V would still be multiplied by a weight of 0.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

struct jg_kvq {
  jg_dev* dev;
  jg_kvcache_desc d;
  int format;
  uint8_t* k_codes;  // [L][n_pages][G][page][hd]
  uint8_t* v_codes;
  __half2* scales;   // [L][n_pages][G][page], (K, V)
  int32_t* block_table;
  int max_ctx;
  size_t layer_rows;  // (position, kv head) rows of a layer
  uint64_t bytes;
};

// What the kernels see of one layer.
struct KvqLayer {
  uint8_t* k;
  uint8_t* v;
  __half2* scales;
  const int32_t* block_table;
  int G, page_shift, max_pages, n_seq, max_ctx;
};

static inline KvqLayer kvq_layer(const jg_kvq* kv, int layer) {
  KvqLayer l;
  const size_t rows = kv->layer_rows * layer;
  l.k = kv->k_codes + rows * kv->d.head_dim;
  l.v = kv->v_codes + rows * kv->d.head_dim;
  l.scales = kv->scales + rows;
  l.block_table = kv->block_table;
  l.G = kv->d.n_kv_heads;
  l.page_shift = 0;
  while ((1 << l.page_shift) < kv->d.page_size) l.page_shift++;
  l.max_pages = kv->d.max_pages_per_seq;
  l.n_seq = kv->d.max_batch;
  l.max_ctx = kv->max_ctx;
  return l;
}

#ifdef __CUDACC__
constexpr int KVQ_INT8 = JG_KVQ_INT8, KVQ_E4M3 = JG_KVQ_E4M3;

// Four codes of zeros.  An int8 code lies in the cache as code + 128, which saves what widens it an operation.
template <int FMT>
constexpr uint32_t KVQ_ZERO = FMT == KVQ_INT8 ? 0x80808080u : 0u;

// Row of (position t, kv head g) in a layer's pools, for the sequence with this row of the block table (entries were checked when
// the table was set).
__device__ __forceinline__ size_t kvq_row(const KvqLayer& c, const int32_t* bt_row, int t, int g) {
  return ((((size_t)bt_row[t >> c.page_shift] * c.G + g) << c.page_shift)) + (t & ((1 << c.page_shift) - 1));
}

// Four codes (a word) as two pairs of halves, without their scale.
template <int FMT>
__device__ __forceinline__ void kvq_widen(uint32_t w, __half2& lo, __half2& hi) {
  if (FMT == KVQ_INT8) {
    const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);  // behind the exponent of 1024
    const __half2 bias = __floats2half2_rn(1152.f, 1152.f);
    lo = __hsub2(*reinterpret_cast<const __half2*>(&a), bias);
    hi = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
  } else {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xFFFFu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    lo = *reinterpret_cast<const __half2*>(&a);
    hi = *reinterpret_cast<const __half2*>(&b);
  }
}

// The scale of a row whose largest magnitude is a (finite).  The quotient is a product with a constant that is 2^-20 of itself too
// small: less than a quotient beyond a border is away from it, more than the roundings, so one on a border is rounded up to it.
template <int FMT>
__device__ __forceinline__ float kvq_scale(float a) {
  if (a == 0.f) return 0.f;
  if (FMT == KVQ_INT8) {
    const float s = a * (float)((1.0 - 0x1p-20) / 127.0);
    if (s < 0x1p-21f) return ceilf(s * 0x1p24f) * 0x1p-24f;                // multiples of 2^-24
    return __uint_as_float((__float_as_uint(s) + 0xFFFFFu) & ~0xFFFFFu);  // 3 bits behind the leading one
  }
  const uint32_t s = (__float_as_uint(a * (float)((1.0 - 0x1p-20) / 448.0)) + 0x7FFFFFu) & ~0x7FFFFFu;  // the next power of two
  return fmaxf(__uint_as_float(s), 0x1p-15f);
}
// What a row's values are multiplied by to be codes.
template <int FMT>
__device__ __forceinline__ float kvq_inverse(float scale) {
  if (FMT != KVQ_INT8) return __uint_as_float(0x7F000000u - __float_as_uint(scale));  // 2^-e
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale));  // to 2^-23
  return r;
}
// Eight values as two words of codes.  A scale beyond 512 (from 256 on) has codes whose values pass 65504: the largest that does not is 113 (240).
// int8: the product is off by less than 2^-15 from x / scale, which is at most 127.  A quotient that is no tie is at least 2^-12 away
// from one (x has 11 significant bits, scale 4), so rounding to multiples of 2^-13 first makes ties of the ties and of nothing
// else.  Adding 1536 is that rounding, adding 1.5 2^23 less that the one to whole numbers, and 128 more the code's bias.
template <int FMT>
__device__ __forceinline__ uint2 kvq_codes(float (&x)[8], float scale, float inverse) {
  if (!(scale > 0.f)) return make_uint2(KVQ_ZERO<FMT>, KVQ_ZERO<FMT>);
  if (FMT == KVQ_INT8 ? scale > 512.f : scale >= 256.f) {
    const float top = (FMT == KVQ_INT8 ? 113.f : 240.f) * scale;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = fminf(fmaxf(x[i], -top), top);
  }
  if (FMT == KVQ_INT8) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = __float_as_uint(__fadd_rn(fmaf(x[i], inverse, 1536.f), 12583040.f - 1536.f));
    return make_uint2(__byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(w[4], w[5], 0x0040), __byte_perm(w[6], w[7], 0x0040), 0x5410));
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) w[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i] * inverse, x[2 * i + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

// Eight halves, four pairs, turned by (cos, sin): products of halves are exact in 32 bits, so each value is rounded there once and
// then to half.
__device__ __forceinline__ uint4 kvq_rotate(const uint4& x, const uint4& t) {
  const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ts[4] = {t.x, t.y, t.z, t.w};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 v = h2_to_f2(xs[i]), c = h2_to_f2(ts[i]);
    const __half2 h = __floats2half2_rn(fmaf(v.x, c.x, -(v.y * c.y)), fmaf(v.x, c.y, v.y * c.x));
    o[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// A K and a V row spread over LPR neighbouring lanes, eight values each (K rotated already): their codes and scales.
template <int FMT, int LPR>
__device__ __forceinline__ void kvq_quantise(const uint4& k, const uint4& v, uint2& kc, uint2& vc, __half2& scale) {
  // the largest magnitudes, K's and V's as one pair of halves; a NaN stays
  const auto top = [](const uint4& v) {
    const uint32_t w[4] = {v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu, v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu};
    const __half2* h = reinterpret_cast<const __half2*>(w);
    return __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
  };
  const __half2 tk = top(k), tv = top(v);
  __half2 t = __hmax2_nan(__lows2half2(tk, tv), __highs2half2(tk, tv));
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<const uint32_t*>(&t), o);
    t = __hmax2_nan(t, *reinterpret_cast<const __half2*>(&other));
  }
  const float a = __low2float(t), b = __high2float(t);
  if (!(a <= 65504.f) || !(b <= 65504.f)) {
    kc = vc = make_uint2(KVQ_ZERO<FMT>, KVQ_ZERO<FMT>);
    scale = __halves2half2(__ushort_as_half(0x7FFF), __ushort_as_half(0));
    return;
  }
  float x[8], y[8];
  unpack8(k, x);
  unpack8(v, y);
  const float sk = kvq_scale<FMT>(a), sv = kvq_scale<FMT>(b), ik = kvq_inverse<FMT>(sk), iv = kvq_inverse<FMT>(sv);
  kc = kvq_codes<FMT>(x, sk, ik);
  vc = kvq_codes<FMT>(y, sv, iv);
  scale = __floats2half2_rn(sk, sv);
}
#endif
