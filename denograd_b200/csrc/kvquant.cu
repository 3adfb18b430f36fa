// The 8-bit KV cache: the object, storing new rows (RoPE, quantisation) and reading them back.  What attends to it: kvquant_attn.cu.
#include <stdlib.h>
#include <string.h>

#include <mutex>
#include <new>

#include "kvquant_chunk.cuh"
#include "kvquant_split.cuh"

// ------------------------------------------------------------------------------------------------ the object
// The device's workspace for results that several CTAs share, for either kernel and any cache.
static int kvq_workspace(jg_dev* dev) {
  static std::mutex m;
  std::lock_guard<std::mutex> lock(m);
  if (dev->kvq_part != nullptr) return JG_OK;
  const size_t few = (size_t)ks_slots(dev) * ks_part_floats(128), many = (size_t)kc_slots(dev) * kc_part_floats(128);
  const size_t part = (few > many ? few : many) * sizeof(float), tickets = jg_kvq_ticket_bytes(dev);
  void* p = nullptr;
  JG_CUDA(cudaMalloc(&p, part + tickets));
  const cudaError_t e = cudaMemsetAsync((char*)p + part, 0, tickets, dev->stream);
  if (e != cudaSuccess) { cudaFree(p); return jg_cuda_fail(e, "kvq workspace", __FILE__, __LINE__); }
  dev->kvq_tickets = (unsigned int*)((char*)p + part);
  dev->kvq_part = (float*)p;
  return JG_OK;
}

JG_API int jg_kvq_create(jg_dev* dev, const jg_kvcache_desc* desc, int32_t format, jg_kvq** out) {
  JG_ENTER(dev);
  JG_REQUIRE(desc != nullptr && out != nullptr, "kvq_create: null argument");
  const jg_kvcache_desc& d = *desc;
  JG_REQUIRE(format == JG_KVQ_INT8 || format == JG_KVQ_E4M3, "kvq_create: unknown format %d", format);
  JG_REQUIRE(d.n_layers > 0 && d.n_kv_heads > 0 && d.n_pages > 0 && d.max_batch > 0 && d.max_pages_per_seq > 0 && d.n_heads > 0,
             "kvq_create: non-positive dimension");
  JG_REQUIRE(d.head_dim == 64 || d.head_dim == 128, "kvq_create: head_dim %d not supported (64 or 128)", d.head_dim);
  JG_REQUIRE(d.page_size == 16 || d.page_size == 32 || d.page_size == 64, "kvq_create: page_size %d not in {16,32,64}", d.page_size);
  JG_REQUIRE(d.n_heads % d.n_kv_heads == 0 && d.n_heads / d.n_kv_heads <= 8,
             "kvq_create: %d query heads for %d kv heads: 1 to 8 to each are supported", d.n_heads, d.n_kv_heads);
  // what 32-bit indexes hold: query rows of a chunk, tiles of an item's heads, rows of a layer's pool
  JG_REQUIRE(d.n_heads <= 4096, "kvq_create: %d heads", d.n_heads);
  JG_REQUIRE((long long)d.max_batch * d.max_pages_per_seq <= 0x7fffffffLL && (long long)d.max_pages_per_seq * d.page_size <= (1 << 24),
             "kvq_create: block table too large, or more than 2^24 positions to a slot");
  JG_REQUIRE((unsigned long long)d.n_pages * d.n_kv_heads * d.page_size <= 0xffffffffull, "kvq_create: pool too large");
  JG_REQUIRE(!dev->capturing, "kvq_create: a graph capture is in progress");
  const int rc = kvq_workspace(dev);
  if (rc) return rc;
  jg_kvq* kv = new (std::nothrow) jg_kvq();
  JG_REQUIRE(kv != nullptr, "kvq_create: out of memory");
  kv->dev = dev;
  kv->d = d;
  kv->format = format;
  kv->max_ctx = d.max_pages_per_seq * d.page_size;
  kv->layer_rows = (size_t)d.n_pages * d.n_kv_heads * d.page_size;
  const size_t rows = kv->layer_rows * d.n_layers, codes = rows * d.head_dim, table = (size_t)d.max_batch * d.max_pages_per_seq * sizeof(int32_t);
  cudaError_t e = cudaMalloc(&kv->k_codes, codes);
  if (e == cudaSuccess) e = cudaMalloc(&kv->v_codes, codes);
  if (e == cudaSuccess) e = cudaMalloc(&kv->scales, rows * sizeof(__half2));
  if (e == cudaSuccess) e = cudaMalloc(&kv->block_table, table);
  int32_t* ids = (int32_t*)malloc(table);
  if (e == cudaSuccess && ids == nullptr) e = cudaErrorMemoryAllocation;
  if (e == cudaSuccess) {
    // zeros, as a new fp16 cache has (positions nobody wrote are read behind masks); row b of the block table owns pages
    // [b * max_pages_per_seq, ...) as far as the pool reaches
    for (int b = 0; b < d.max_batch; b++)
      for (int i = 0; i < d.max_pages_per_seq; i++) {
        const long long pg = (long long)b * d.max_pages_per_seq + i;
        ids[(size_t)b * d.max_pages_per_seq + i] = (int32_t)(pg < d.n_pages ? pg : d.n_pages - 1);
      }
    const int zero = format == JG_KVQ_INT8 ? 128 : 0;
    e = cudaMemsetAsync(kv->k_codes, zero, codes, dev->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(kv->v_codes, zero, codes, dev->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(kv->scales, 0, rows * sizeof(__half2), dev->stream);
    if (e == cudaSuccess) e = cudaMemcpyAsync(kv->block_table, ids, table, cudaMemcpyHostToDevice, dev->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(dev->stream);
  }
  free(ids);
  if (e != cudaSuccess) {
    cudaGetLastError();
    jg_kvq_destroy(kv);
    return jg_cuda_fail(e, "kvq_create", __FILE__, __LINE__);
  }
  kv->bytes = 2 * codes + rows * sizeof(__half2) + table;
  *out = kv;
  return JG_OK;
}

static void kvq_destroy_now(void* p) { jg_kvq_destroy((jg_kvq*)p); }

JG_API int jg_kvq_destroy(jg_kvq* kv) {
  if (!kv) return JG_OK;
  if (g_jg_capturing > 0) { jg_defer(kvq_destroy_now, kv); return JG_OK; }
  cudaSetDevice(kv->dev->ordinal);
  cudaStreamSynchronize(kv->dev->stream);
  cudaFree(kv->k_codes); cudaFree(kv->v_codes); cudaFree(kv->scales); cudaFree(kv->block_table);
  delete kv;
  return JG_OK;
}

JG_API int jg_kvq_set_block_table(jg_kvq* kv, const int32_t* table) {
  JG_REQUIRE(kv != nullptr && table != nullptr, "kvq_set_block_table: null argument");
  JG_ENTER(kv->dev);
  JG_REQUIRE(!kv->dev->capturing, "kvq_set_block_table: a graph capture is in progress");
  const size_t n = (size_t)kv->d.max_batch * kv->d.max_pages_per_seq;
  for (size_t i = 0; i < n; i++)
    JG_REQUIRE(table[i] >= 0 && table[i] < kv->d.n_pages, "kvq_set_block_table: entry %zu = %d outside the pool of %d pages", i, table[i], kv->d.n_pages);
  JG_CUDA(cudaMemcpyAsync(kv->block_table, table, n * sizeof(int32_t), cudaMemcpyHostToDevice, kv->dev->stream));
  JG_CUDA(cudaStreamSynchronize(kv->dev->stream));
  return JG_OK;
}

JG_API int jg_kvq_bytes(jg_kvq* kv, uint64_t* out) {
  JG_REQUIRE(kv != nullptr && out != nullptr, "kvq_bytes: null argument");
  *out = kv->bytes;
  return JG_OK;
}

// ------------------------------------------------------------------------------------------------ storing
struct KvqWriteArgs {
  KvqLayer c;
  __half* q_out;
  const __half* qkv;
  const __half* table;  // [table_rows][hd/2][2], or null
  const int32_t* pos;
  const int32_t* seq;
  int ldq, ldx, table_rows, R, H;
};

constexpr int KW_THREADS = 128;

// A thread for each eight values of a row's Q heads, and of its K heads together with V, of U neighbouring rows: all their loads
// are on their way before any is waited for (positions and slots are not needed for the values, only for where they go).
// Bound by its passes over rows and codes: 3800 rows of the 8B, 86 MB with the rotated queries, 18.7 us, 4.6 TB/s; issue slots are 70 % busy.
template <int FMT, int HD, int U>
__global__ void __launch_bounds__(KW_THREADS) kvq_write_kernel(const KvqWriteArgs a) {
  constexpr int LPR = HD / 8;
  pdl_launch();
  pdl_wait();
  const unsigned per_row = (unsigned)(a.H + a.c.G) * LPR, at = blockIdx.x * (unsigned)KW_THREADS + threadIdx.x, group = at / per_row;
  const int piece = (int)(at - group * per_row), head = piece / LPR, sub = piece % LPR;
  const bool is_q = head < a.H;
  const int row0 = (int)group * U;
  uint4 v[U], w[U], turn[U];
  int t[U], sq[U];
#pragma unroll
  for (int k = 0; k < U; k++) {
    const bool in = row0 + k < a.R;
    const __half* x = a.qkv + (size_t)(in ? row0 + k : 0) * a.ldx + (size_t)head * HD + sub * 8;
    t[k] = in ? a.pos[row0 + k] : -1;
    sq[k] = in ? (a.seq ? a.seq[row0 + k] : row0 + k) : -1;
    v[k] = w[k] = turn[k] = make_uint4(0, 0, 0, 0);
    if (in && (!is_q || a.q_out)) v[k] = ld_128(x);
    if (in && !is_q) w[k] = ld_128(x + (size_t)a.c.G * HD);
  }
#pragma unroll
  for (int k = 0; k < U; k++) {
    if ((unsigned)sq[k] >= (unsigned)a.c.n_seq || (unsigned)t[k] >= (unsigned)a.c.max_ctx || (a.table && t[k] >= a.table_rows)) t[k] = -1;
    if (a.table && t[k] >= 0) turn[k] = ld_128(a.table + (size_t)t[k] * HD + sub * 8);
  }
  size_t to[U];
#pragma unroll
  for (int k = 0; k < U; k++) to[k] = !is_q && t[k] >= 0 ? kvq_row(a.c, a.c.block_table + (size_t)sq[k] * a.c.max_pages, t[k], head - a.H) : 0;
#pragma unroll
  for (int k = 0; k < U; k++) {
    if (a.table) v[k] = kvq_rotate(v[k], turn[k]);
    if (is_q && a.q_out && t[k] >= 0) *reinterpret_cast<uint4*>(a.q_out + (size_t)(row0 + k) * a.ldq + (size_t)head * HD + sub * 8) = v[k];
    if (__all_sync(0xffffffffu, is_q || t[k] < 0)) continue;
    uint2 kc, vc;
    __half2 scale;
    kvq_quantise<FMT, LPR>(v[k], w[k], kc, vc, scale);
    if (!is_q && t[k] >= 0) {
      *reinterpret_cast<uint2*>(a.c.k + to[k] * HD + sub * 8) = kc;
      *reinterpret_cast<uint2*>(a.c.v + to[k] * HD + sub * 8) = vc;
      if (sub == 0) a.c.scales[to[k]] = scale;
    }
  }
}

template <int FMT, int HD>
static int launch_write(jg_dev* dev, const KvqWriteArgs& a) {
  // Two rows to a thread where that leaves every SM sixteen CTAs; below, one.  3800 rows of the 8B: 20.3 us with one, 19.4 with two, 21.3
  // with four (registers: fewer warps); 18.7 with CTAs of 128, 22.5 of 64.
  const unsigned long long per_row = (unsigned long long)(a.H + a.c.G) * (HD / 8), two = ((a.R + 1) / 2 * per_row + KW_THREADS - 1) / KW_THREADS;
  if (two >= 16ull * dev->sm_count) return jg_launch(dev, "kvq_write", kvq_write_kernel<FMT, HD, 2>, dim3((unsigned)two), dim3(KW_THREADS), 0, a);
  return jg_launch(dev, "kvq_write", kvq_write_kernel<FMT, HD, 1>, dim3((unsigned)((a.R * per_row + KW_THREADS - 1) / KW_THREADS)), dim3(KW_THREADS), 0, a);
}

JG_API int jg_kvq_write(jg_dev* dev, jg_kvq* kv, int32_t layer, uint64_t q_out, int32_t ldq, uint64_t qkv, int32_t ldx, uint64_t table,
                        int32_t table_rows, uint64_t pos, uint64_t seq, int32_t R, int32_t H) {
  JG_ENTER(dev);
  JG_REQUIRE(kv != nullptr && kv->dev == dev, "kvq_write: cache belongs to another device");
  JG_REQUIRE(layer >= 0 && layer < kv->d.n_layers, "kvq_write: layer %d out of range", layer);
  const int G = kv->d.n_kv_heads, hd = kv->d.head_dim;
  JG_REQUIRE(H == kv->d.n_heads, "kvq_write: H=%d does not match the cache (n_heads %d)", H, kv->d.n_heads);
  JG_REQUIRE(R > 0 && (seq != 0 || R <= kv->d.max_batch), "kvq_write: R=%d rows for %d slots", R, kv->d.max_batch);
  JG_REQUIRE(ldx >= (H + 2 * G) * hd && ldx % 8 == 0, "kvq_write: rows of %d elements are no multiple of 8 or too short", ldx);
  JG_REQUIRE(q_out == 0 || (ldq >= H * hd && ldq % 8 == 0), "kvq_write: rows of q_out of %d elements are no multiple of 8 or too short", ldq);
  JG_REQUIRE(jg_aligned(qkv, 16) && q_out % 16 == 0 && table % 16 == 0 && jg_aligned(pos, 4) && seq % 4 == 0, "kvq_write: null or misaligned pointer");
  JG_REQUIRE(table == 0 || table_rows > 0, "kvq_write: empty RoPE table");
  const unsigned long long pieces = (unsigned long long)R * (H + G) * (hd / 8);
  JG_REQUIRE(pieces <= 0xffffff00ull, "kvq_write: %d rows are too many for one call", R);
  KvqWriteArgs a = {};
  a.c = kvq_layer(kv, layer);
  a.q_out = (__half*)q_out; a.qkv = (const __half*)qkv; a.table = (const __half*)table;
  a.pos = (const int32_t*)pos; a.seq = (const int32_t*)seq;
  a.ldq = ldq; a.ldx = ldx; a.table_rows = table_rows; a.R = R; a.H = H;
  if (q_out) jg_mark_fresh(dev, q_out, (uint64_t)R * ldq * 2);  // what is written may be the next call's weight matrix, here and below
  if (kv->format == JG_KVQ_INT8) return hd == 64 ? launch_write<KVQ_INT8, 64>(dev, a) : launch_write<KVQ_INT8, 128>(dev, a);
  return hd == 64 ? launch_write<KVQ_E4M3, 64>(dev, a) : launch_write<KVQ_E4M3, 128>(dev, a);
}

// ------------------------------------------------------------------------------------------------ reading back
struct KvqReadArgs {
  KvqLayer c;
  __half* k;
  __half* v;
  const int32_t* pos;
  const int32_t* count;
  const int32_t* first;
  const int32_t* seq;
  int ld, R, max_count, step;
};

constexpr int KR_THREADS = 256, KR_ROWS = 4;

// A thread for each eight values of K and the eight of V beside them, of U neighbouring positions, whose loads are in flight together (8 ragged
// stretches, 8B: 18 us with two positions to a thread, 10.3 with four, 44 MB at 4.3 TB/s; even ones, 201 MB, 35.2 us, 5.7 TB/s).
template <int FMT, int HD>
__global__ void __launch_bounds__(KR_THREADS) kvq_read_kernel(const KvqReadArgs a) {
  constexpr int LPR = HD / 8, U = KR_ROWS;
  pdl_launch();
  pdl_wait();
  const int b = blockIdx.y;
  const unsigned per_row = (unsigned)a.c.G * LPR;
  const int count = a.count ? a.count[b] : a.max_count, first = a.first ? a.first[b] : b, p0 = a.pos[b], sq = a.seq ? a.seq[b] : b;
  const int n = min(count, a.max_count);
  const bool known = (unsigned)sq < (unsigned)a.c.n_seq;
  const int32_t* bt_row = a.c.block_table + (size_t)(known ? sq : 0) * a.c.max_pages;
  for (unsigned at = blockIdx.x * KR_THREADS + threadIdx.x;; at += gridDim.x * KR_THREADS) {  // below 2^31: see the limit of a call
    const unsigned group = at / per_row;
    const long long i0 = (long long)group * U;
    if (i0 >= n) return;
    const int piece = (int)(at - group * per_row), g = piece / LPR, sub = piece % LPR;
    size_t from[U];
    bool live[U];
#pragma unroll
    for (int k = 0; k < U; k++) {
      const long long t = p0 + i0 + k;
      live[k] = known && i0 + k < n && t >= 0 && t < a.c.max_ctx;
      from[k] = live[k] ? kvq_row(a.c, bt_row, (int)t, g) : 0;
    }
    uint2 kc[U], vc[U];
    __half2 scale[U];
#pragma unroll
    for (int k = 0; k < U; k++) {
      kc[k] = vc[k] = make_uint2(KVQ_ZERO<FMT>, KVQ_ZERO<FMT>);
      scale[k] = __half2half2(__ushort_as_half(0));
      if (live[k]) {
        kc[k] = *reinterpret_cast<const uint2*>(a.c.k + from[k] * HD + sub * 8);
        vc[k] = *reinterpret_cast<const uint2*>(a.c.v + from[k] * HD + sub * 8);
        scale[k] = a.c.scales[from[k]];
      }
    }
#pragma unroll
    for (int k = 0; k < U; k++) {
      const long long row = first + (i0 + k) * a.step;
      if (i0 + k >= n || row < 0 || row >= a.R) continue;
      const __half2 sk = __low2half2(scale[k]), sv = __hisnan(__low2half(scale[k])) ? sk : __high2half2(scale[k]);
      __half2 h[4], w[4];
      kvq_widen<FMT>(kc[k].x, h[0], h[1]);
      kvq_widen<FMT>(kc[k].y, h[2], h[3]);
      kvq_widen<FMT>(vc[k].x, w[0], w[1]);
      kvq_widen<FMT>(vc[k].y, w[2], w[3]);
#pragma unroll
      for (int j = 0; j < 4; j++) { h[j] = __hmul2_rn(h[j], sk); w[j] = __hmul2_rn(w[j], sv); }
      const size_t to = (size_t)row * a.ld + (size_t)g * HD + sub * 8;
      *reinterpret_cast<uint4*>(a.k + to) = *reinterpret_cast<const uint4*>(h);
      *reinterpret_cast<uint4*>(a.v + to) = *reinterpret_cast<const uint4*>(w);
    }
  }
}

template <int FMT, int HD>
static int launch_read(jg_dev* dev, const KvqReadArgs& a, int B) {
  const unsigned long long per_row = (unsigned long long)a.c.G * (HD / 8), ctas = ((a.max_count + KR_ROWS - 1) / KR_ROWS * per_row + KR_THREADS - 1) / KR_THREADS;
  // A ragged batch has many CTAs without rows: 5, 10, 20 an SM, and one for each piece 14.9, 12.3, 10.3, 11.4 us.
  const unsigned long long most = (20ull * dev->sm_count + B - 1) / B;
  return jg_launch(dev, "kvq_read", kvq_read_kernel<FMT, HD>, dim3((unsigned)(ctas < most ? ctas : most), (unsigned)B), dim3(KR_THREADS), 0, a);
}

JG_API int jg_kvq_read(jg_dev* dev, jg_kvq* kv, int32_t layer, uint64_t k, uint64_t v, int32_t ld, int32_t R, uint64_t pos, uint64_t count,
                       uint64_t first, uint64_t seq, int32_t B, int32_t max_count, int32_t step) {
  JG_ENTER(dev);
  JG_REQUIRE(kv != nullptr && kv->dev == dev, "kvq_read: cache belongs to another device");
  JG_REQUIRE(layer >= 0 && layer < kv->d.n_layers, "kvq_read: layer %d out of range", layer);
  const int G = kv->d.n_kv_heads, hd = kv->d.head_dim;
  JG_REQUIRE(R > 0 && max_count > 0 && max_count <= kv->max_ctx && step > 0 && B > 0 && B <= 65535 && (seq != 0 || B <= kv->d.max_batch),
             "kvq_read: B=%d sequences of up to %d positions, R=%d rows, %d slots", B, max_count, R, kv->d.max_batch);
  JG_REQUIRE(ld >= G * hd && ld % 8 == 0, "kvq_read: rows of %d elements are no multiple of 8 or too short", ld);
  JG_REQUIRE(jg_aligned(k, 16) && jg_aligned(v, 16) && jg_aligned(pos, 4) && count % 4 == 0 && first % 4 == 0 && seq % 4 == 0, "kvq_read: null or misaligned pointer");
  const unsigned long long pieces = (unsigned long long)max_count * G * (hd / 8);
  JG_REQUIRE(pieces <= 0xffffff00ull, "kvq_read: %d positions are too many for one call", max_count);
  KvqReadArgs a = {};
  a.c = kvq_layer(kv, layer);
  a.k = (__half*)k; a.v = (__half*)v;
  a.pos = (const int32_t*)pos; a.count = (const int32_t*)count; a.first = (const int32_t*)first; a.seq = (const int32_t*)seq;
  a.ld = ld; a.R = R; a.max_count = max_count; a.step = step;
  jg_mark_fresh(dev, k, (uint64_t)R * ld * 2);
  jg_mark_fresh(dev, v, (uint64_t)R * ld * 2);
  if (kv->format == JG_KVQ_INT8) return hd == 64 ? launch_read<KVQ_INT8, 64>(dev, a, B) : launch_read<KVQ_INT8, 128>(dev, a, B);
  return hd == 64 ? launch_read<KVQ_E4M3, 64>(dev, a, B) : launch_read<KVQ_E4M3, 128>(dev, a, B);
}
