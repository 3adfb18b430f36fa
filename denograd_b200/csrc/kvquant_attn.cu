// Attention over the 8-bit KV cache: one new token a row (jg_kvq_decode) and chunks (jg_kvq_attn).
//
// Few queries to a (sequence, kv head) go to the kernel that is bound by reading the cache (kvquant_split.cuh), more to the one on the 5th-generation
// tensor cores (kvquant_chunk.cu).  Both compute o = sum_t w_t v_t / sum_t w_t with w_t = e^(s_t - max), s_t = q.k_t / sqrt(hd), in one pass with a
// running maximum; w is rounded to fp16 for the product with V and summed as it was.
#include <math.h>

#include "kvquant_chunk.cuh"
#include "kvquant_split.cuh"

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
  a.part = dev->kvq_part; a.tickets = dev->kvq_tickets;
  jg_mark_fresh(dev, out, (uint64_t)B * ldo * 2);  // may be the next call's weight matrix
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
  JG_REQUIRE(R > 0 && max_count > 0 && max_count <= kv->max_ctx && step > 0 && B > 0 && B <= 65535 && (seq != 0 || B <= kv->d.max_batch),
             "kvq_attn: B=%d sequences of up to %d positions, R=%d rows, %d slots", B, max_count, R, kv->d.max_batch);
  JG_REQUIRE(ldq >= H * hd && ldq % 8 == 0 && ldo >= H * hd && ldo % 8 == 0, "kvq_attn: rows of %d and %d elements are no multiple of 8 or too short", ldq, ldo);
  JG_REQUIRE(jg_aligned(out, 16) && jg_aligned(q, 16) && jg_aligned(pos, 4) && count % 4 == 0 && first % 4 == 0 && seq % 4 == 0, "kvq_attn: null or misaligned pointer");
  jg_mark_fresh(dev, out, (uint64_t)R * ldo * 2);
  // Few columns are read at HBM's pace or near it: 8 sequences behind 3001 positions of the 8B, 16 columns 24.8 us (the tensor cores' form 37.7), 20
  // columns 28.6 (37.7), 24 columns 28.7 (37.7), 32 sequences of 20 columns 71 (96); 24 sequences behind 4000 of the 1B, 28 columns 56 (75).  A lane's
  // outputs have to fit its registers: 32 columns of 128 values would take 42 us, against 38.
  if ((long long)max_count * (H / G) <= (hd == 64 ? 32 : 24)) {
    KvqSplitArgs s = {};
    s.c = kvq_layer(kv, layer);
    s.x = (const __half*)q; s.out = (__half*)out;
    s.pos = (const int32_t*)pos; s.count = (const int32_t*)count; s.first = (const int32_t*)first; s.seq = (const int32_t*)seq;
    s.ldx = ldq; s.ldo = ldo; s.R = R; s.B = B; s.H = H; s.n_rep = H / G; s.max_count = max_count; s.step = step;
    s.limit = kv->max_ctx;
    s.scale2 = (float)(1.4426950408889634 / sqrt((double)hd));
    s.part = dev->kvq_part; s.tickets = dev->kvq_tickets;
    const int columns = max_count * (H / G);
#define KS_CASE(FMT_, FORMAT_, HD_)                                                      \
  if (kv->format == FORMAT_ && hd == HD_)                                                \
    return columns <= 8    ? launch_split<FMT_, HD_, 1, false>(dev, s)                   \
           : columns <= 16 ? launch_split<FMT_, HD_, 2, false>(dev, s)                   \
           : columns <= 24 ? launch_split<FMT_, HD_, 3, false>(dev, s)                   \
                           : launch_split<FMT_, HD_, HD_ == 64 ? 4 : 3, false>(dev, s);
    KS_CASE(KVQ_INT8, JG_KVQ_INT8, 64) KS_CASE(KVQ_INT8, JG_KVQ_INT8, 128) KS_CASE(KVQ_E4M3, JG_KVQ_E4M3, 64) KS_CASE(KVQ_E4M3, JG_KVQ_E4M3, 128)
#undef KS_CASE
  }
  KvqChunkArgs a = {};
  a.c = kvq_layer(kv, layer);
  a.q = (const __half*)q; a.out = (__half*)out;
  a.pos = (const int32_t*)pos; a.count = (const int32_t*)count; a.first = (const int32_t*)first; a.seq = (const int32_t*)seq;
  a.ldq = ldq; a.ldo = ldo; a.R = R; a.B = B; a.n_rep = H / G; a.max_count = max_count; a.step = step;
  a.max_tiles = (int)(((long long)max_count * (H / G) + KC_ROWS - 1) / KC_ROWS);
  JG_REQUIRE((long long)B * a.max_tiles <= (1 << 26), "kvq_attn: B=%d sequences of up to %d positions are too many for one call", B, max_count);
  a.scale2 = (float)(1.4426950408889634 / sqrt((double)hd));
  a.part = dev->kvq_part; a.tickets = dev->kvq_tickets; a.err = dev->err_word;
  return kvq_chunk(dev, kv->format, hd, a);
}
