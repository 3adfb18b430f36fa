// Attention over the 8-bit KV cache: one new token a row (jg_kvq_decode) and chunks (jg_kvq_attn).
//
// o = sum_t w_t v_t / sum_t w_t with w_t = 2^((s_t - max) / ln 2), s_t = q.k_t / sqrt(hd), in one pass over the cache with a running maximum.
#include <math.h>

#include "kvquant_split.cuh"

struct KvqAttnArgs {
  KvqLayer c;
  const __half* q;
  __half* out;
  const int32_t* pos;
  const int32_t* count;
  const int32_t* first;
  const int32_t* seq;
  int ldq, ldo, R, H, n_rep, max_count, step;
  int table_rows;  // positions from here on are outside too (decode with a RoPE table); max_ctx otherwise
  float scale2;    // log2 e / sqrt(hd)
};

constexpr int KA_THREADS = 128;

// A warp for each query head of a (position, kv head); lanes hold hd / 32 neighbouring values.
template <int FMT, int HD>
__global__ void __launch_bounds__(KA_THREADS) kvq_attn_kernel(const KvqAttnArgs a) {
  constexpr int V = HD / 32;
  pdl_launch();
  pdl_wait();
  const int i = blockIdx.x, g = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = a.count ? min(a.count[b], a.max_count) : a.max_count;
  if (i >= n) return;
  const long long row = (long long)(a.first ? a.first[b] : b) + (long long)i * a.step, last = (long long)a.pos[b] + i;
  if (row < 0 || row >= a.R) return;
  const int sq = a.seq ? a.seq[b] : b;
  const bool live = (unsigned)sq < (unsigned)a.c.n_seq && last >= 0 && last < a.table_rows;
  const int32_t* bt_row = a.c.block_table + (size_t)(live ? sq : 0) * a.c.max_pages;
  for (int h = warp; h < a.n_rep; h += KA_THREADS / 32) {
    const size_t col = (size_t)(g * a.n_rep + h) * HD + lane * V;
    float q[V], o[V], m = -INFINITY, l = 0.f;
    for (int j = 0; j < V; j++) { q[j] = __half2float(a.q[(size_t)row * a.ldq + col + j]); o[j] = 0.f; }
    for (int t = 0; live && t <= (int)last; t++) {
      const size_t at = kvq_row(a.c, bt_row, t, g);
      uint32_t kw, vw;
      if (V == 4) {
        kw = *reinterpret_cast<const uint32_t*>(a.c.k + at * HD + lane * V);
        vw = *reinterpret_cast<const uint32_t*>(a.c.v + at * HD + lane * V);
      } else {
        kw = *reinterpret_cast<const uint16_t*>(a.c.k + at * HD + lane * V);
        vw = *reinterpret_cast<const uint16_t*>(a.c.v + at * HD + lane * V);
      }
      const float2 sc = __half22float2(a.c.scales[at]);
      __half2 k[2], v[2];
      kvq_widen<FMT>(kw, k[0], k[1]);
      kvq_widen<FMT>(vw, v[0], v[1]);
      const float kf[4] = {__low2float(k[0]), __high2float(k[0]), __low2float(k[1]), __high2float(k[1])};
      const float vf[4] = {__low2float(v[0]), __high2float(v[0]), __low2float(v[1]), __high2float(v[1])};
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < V; j++) s = fmaf(q[j], kf[j] * sc.x, s);
      s = warp_sum(s) * a.scale2;
      const float top = fmaxf(m, s), fade = exp2f(m - top), w = exp2f(s - top);
      l = fmaf(l, fade, w);
#pragma unroll
      for (int j = 0; j < V; j++) o[j] = fmaf(o[j], fade, w * (vf[j] * sc.y));
      m = top;
    }
    for (int j = 0; j < V; j++) a.out[(size_t)row * a.ldo + col + j] = __float2half_rn(live ? __fdiv_rn(o[j], l) : 0.f);
  }
}

static int launch_attn(jg_dev* dev, const jg_kvq* kv, const KvqAttnArgs& a, int B, const char* what) {
  const dim3 grid((unsigned)a.max_count, (unsigned)kv->d.n_kv_heads, (unsigned)B), block(KA_THREADS);
  if (kv->format == JG_KVQ_INT8)
    return kv->d.head_dim == 64 ? jg_launch(dev, what, kvq_attn_kernel<KVQ_INT8, 64>, grid, block, 0, a)
                                : jg_launch(dev, what, kvq_attn_kernel<KVQ_INT8, 128>, grid, block, 0, a);
  return kv->d.head_dim == 64 ? jg_launch(dev, what, kvq_attn_kernel<KVQ_E4M3, 64>, grid, block, 0, a)
                              : jg_launch(dev, what, kvq_attn_kernel<KVQ_E4M3, 128>, grid, block, 0, a);
}

JG_API int jg_kvq_decode(jg_dev* dev, jg_kvq* kv, int32_t layer, uint64_t out, int32_t ldo, uint64_t qkv, int32_t ldx, uint64_t table,
                         int32_t table_rows, uint64_t pos, uint64_t seq, int32_t B, int32_t H) {
  JG_ENTER(dev);
  JG_REQUIRE(kv != nullptr && kv->dev == dev, "kvq_decode: cache belongs to another device");
  JG_REQUIRE(layer >= 0 && layer < kv->d.n_layers, "kvq_decode: layer %d out of range", layer);
  const int G = kv->d.n_kv_heads, hd = kv->d.head_dim;
  JG_REQUIRE(H == kv->d.n_heads, "kvq_decode: H=%d does not match the cache (n_heads %d)", H, kv->d.n_heads);
  JG_REQUIRE(B > 0 && B <= 65535 && (seq != 0 || B <= kv->d.max_batch), "kvq_decode: B=%d rows for %d slots", B, kv->d.max_batch);
  JG_REQUIRE(ldx >= (H + 2 * G) * hd && ldx % 8 == 0, "kvq_decode: rows of %d elements are no multiple of 8 or too short", ldx);
  JG_REQUIRE(ldo >= H * hd && ldo % 8 == 0, "kvq_decode: rows of out of %d elements are no multiple of 8 or too short", ldo);
  JG_REQUIRE(jg_aligned(out, 16) && jg_aligned(qkv, 16) && table % 16 == 0 && jg_aligned(pos, 4) && seq % 4 == 0, "kvq_decode: null or misaligned pointer");
  JG_REQUIRE(table == 0 || table_rows > 0, "kvq_decode: empty RoPE table");
  KvqSplitArgs a = {};
  a.c = kvq_layer(kv, layer);
  a.x = (const __half*)qkv; a.table = (const __half*)table; a.out = (__half*)out; a.pos = (const int32_t*)pos; a.seq = (const int32_t*)seq;
  a.ldx = ldx; a.ldo = ldo; a.R = B; a.B = B; a.H = H; a.n_rep = H / G; a.max_count = 1; a.step = 1;
  a.limit = table && table_rows < kv->max_ctx ? table_rows : kv->max_ctx;
  a.scale2 = (float)(1.4426950408889634 / sqrt((double)hd));
  a.part = kv->part; a.tickets = kv->tickets;
  if (kv->format == JG_KVQ_INT8) return hd == 64 ? launch_split<KVQ_INT8, 64, 1, true>(dev, a) : launch_split<KVQ_INT8, 128, 1, true>(dev, a);
  return hd == 64 ? launch_split<KVQ_E4M3, 64, 1, true>(dev, a) : launch_split<KVQ_E4M3, 128, 1, true>(dev, a);
}

JG_API int jg_kvq_attn(jg_dev* dev, jg_kvq* kv, int32_t layer, uint64_t out, int32_t ldo, uint64_t q, int32_t ldq, int32_t R, uint64_t pos,
                       uint64_t count, uint64_t first, uint64_t seq, int32_t B, int32_t max_count, int32_t step, int32_t H) {
  JG_ENTER(dev);
  JG_REQUIRE(kv != nullptr && kv->dev == dev, "kvq_attn: cache belongs to another device");
  JG_REQUIRE(layer >= 0 && layer < kv->d.n_layers, "kvq_attn: layer %d out of range", layer);
  const int G = kv->d.n_kv_heads, hd = kv->d.head_dim;
  JG_REQUIRE(H == kv->d.n_heads, "kvq_attn: H=%d does not match the cache (n_heads %d)", H, kv->d.n_heads);
  JG_REQUIRE(R > 0 && max_count > 0 && B > 0 && B <= 65535 && (seq != 0 || B <= kv->d.max_batch), "kvq_attn: B=%d sequences of up to %d positions, R=%d rows, %d slots", B,
             max_count, R, kv->d.max_batch);
  JG_REQUIRE(ldq >= H * hd && ldq % 8 == 0 && ldo >= H * hd && ldo % 8 == 0, "kvq_attn: rows of %d and %d elements are no multiple of 8 or too short", ldq, ldo);
  JG_REQUIRE(jg_aligned(out, 16) && jg_aligned(q, 16) && jg_aligned(pos, 4) && count % 4 == 0 && first % 4 == 0 && seq % 4 == 0, "kvq_attn: null or misaligned pointer");
  if ((long long)max_count * (H / G) <= 16) {
    KvqSplitArgs s = {};
    s.c = kvq_layer(kv, layer);
    s.x = (const __half*)q; s.out = (__half*)out;
    s.pos = (const int32_t*)pos; s.count = (const int32_t*)count; s.first = (const int32_t*)first; s.seq = (const int32_t*)seq;
    s.ldx = ldq; s.ldo = ldo; s.R = R; s.B = B; s.H = H; s.n_rep = H / G; s.max_count = max_count; s.step = step;
    s.limit = kv->max_ctx;
    s.scale2 = (float)(1.4426950408889634 / sqrt((double)hd));
    s.part = kv->part; s.tickets = kv->tickets;
    const bool few = max_count * (H / G) <= 8;
    if (kv->format == JG_KVQ_INT8)
      return hd == 64 ? (few ? launch_split<KVQ_INT8, 64, 1, false>(dev, s) : launch_split<KVQ_INT8, 64, 2, false>(dev, s))
                      : (few ? launch_split<KVQ_INT8, 128, 1, false>(dev, s) : launch_split<KVQ_INT8, 128, 2, false>(dev, s));
    return hd == 64 ? (few ? launch_split<KVQ_E4M3, 64, 1, false>(dev, s) : launch_split<KVQ_E4M3, 64, 2, false>(dev, s))
                    : (few ? launch_split<KVQ_E4M3, 128, 1, false>(dev, s) : launch_split<KVQ_E4M3, 128, 2, false>(dev, s));
  }
  KvqAttnArgs a = {};
  a.c = kvq_layer(kv, layer);
  a.q = (const __half*)q; a.out = (__half*)out;
  a.pos = (const int32_t*)pos; a.count = (const int32_t*)count; a.first = (const int32_t*)first; a.seq = (const int32_t*)seq;
  a.ldq = ldq; a.ldo = ldo; a.R = R; a.H = H; a.n_rep = H / G; a.max_count = max_count; a.step = step;
  a.table_rows = kv->max_ctx;
  a.scale2 = (float)(1.4426950408889634 / sqrt((double)hd));
  return launch_attn(dev, kv, a, B, "kvq_attn");
}
