// Attention of chunks over the 8-bit KV cache on the 5th-generation tensor cores (jg_kvq_attn beyond a few queries).
//
// One pass over the keys with a running maximum: S = Q.K^T, P = 2^(S - m), O += P.V, l += sum P; O / l at the end.  The codes of a tile
// of keys and values become halves, code * scale exactly, on their way into the shared-memory tiles that the products read, so
// a tile crosses HBM as bytes and no 16-bit copy of the cache exists.
//
// A query row is a (position, query head) of one kv head; an item is 256 rows, two streams of 128, over the keys that its last
// row sees, in tiles of 128.  Five warpgroups: softmax of either stream, a thread per row; one that loads and widens K, one for V;
// the last issues the products and keeps the plan.  While one stream's exponentials run, the other's products do; a product with V
// begins when the first half of its weights is there.  Tensor memory: S of both streams (P
// takes its place as 16-bit pairs), O of both.  A row's maximum is a reference that its scores may pass by 2^8 before O is
// rescaled in tensor memory, which is rare behind the first tiles.
//
// The tiles of all items are one line, cut evenly over one CTA for each SM.  An item that several CTAs share meets in a
// workspace; the last to arrive adds the pieces up in order.
//
// What bounds it: per 256 rows x 128 keys x 128 columns four products of 512 cycles at the tensor peak, and 32768
// exponentials at 16 a cycle, 2048 cycles either way; widening takes a fifth of the issue slots beside them.
#include <math.h>

#include "flash_tc.cuh"
#include "kvquant.cuh"
#include "kvquant_chunk.cuh"

// Warps 0-3 and 4-7 softmax, 8-11 keys, 12-15 values, 16 products, 17 plan; 18 and 19 fill up the last warpgroup.
constexpr int KC_THREADS = 640, KC_REGS = 96;                                 // registers at launch
constexpr int KC_SOFT_REGS = 144, KC_WIDEN_REGS = 72, KC_MMA_REGS = 48;       // and from then on, by warpgroup
static_assert(2 * KC_SOFT_REGS + 2 * KC_WIDEN_REGS + KC_MMA_REGS <= 5 * KC_REGS, "register shares exceed what a CTA is launched with");
constexpr int KC_PLAN = 4;  // pieces that the plan is ahead

template <int HD>
struct KcCfg {
  static constexpr uint32_t Q_BYTES = 128 * HD * 2, KV_BYTES = KC_KEYS * HD * 2;
  static constexpr size_t SMEM = 2 * Q_BYTES + 4 * KV_BYTES + 1024;
};

// A piece of work: the key tiles [j0, j1) of an item.
struct KcPiece {
  const int32_t* bt;       // null: the slot lies outside the cache
  int b, tile, g, j0, j1;  // b < 0: no more pieces
  int n_tiles;             // of the whole item
  int p0, n, T;            // first new position and number of new positions of the sequence; keys that the item looks at
  int c_lo, pieces;        // the CTAs that share the item
};

// What a sequence is, and how many key tiles item `tile` of it has (0: no such item).
__device__ __forceinline__ int kc_item(const KvqChunkArgs& a, int b, int tile, KcPiece& p) {
  const int sq = a.seq ? a.seq[b] : b, count = a.count ? a.count[b] : a.max_count;
  p.p0 = a.pos[b];
  p.n = max(0, min(count, a.max_count));
  const int first = a.first ? a.first[b] : b;
  if ((long long)first + (long long)(p.n - 1) * a.step >= a.R) p.n = first < a.R ? (int)(((long long)a.R - 1 - first) / a.step) + 1 : 0;  // rows there are
  if ((long long)tile * KC_ROWS >= (long long)p.n * a.n_rep) return 0;
  const bool have = (unsigned)sq < (unsigned)a.c.n_seq;
  p.bt = have ? a.c.block_table + (size_t)sq * a.c.max_pages : nullptr;
  const int last = min(p.n, ((tile + 1) * KC_ROWS - 1) / a.n_rep + 1);  // positions up to the item's end
  p.T = have ? (int)max(0ll, min((long long)p.p0 + last, (long long)a.c.max_ctx)) : 0;
  return max(1, (p.T + KC_KEYS - 1) / KC_KEYS);
}

// Wait for the loads from tensor memory in flight; nothing that uses their results may move ahead of it.
template <int N>
__device__ __forceinline__ void kc_landed(float* v) {
  tmem_ld_wait();
#pragma unroll
  for (int c = 0; c < N; c++) asm volatile("" : "+f"(v[c]));
}
__device__ __forceinline__ float kc_max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
// the larger of m and v[0 .. N)
template <int N>
__device__ __forceinline__ float kc_max(float m, const float* v) {
  float t0 = m, t1 = v[0];
#pragma unroll
  for (int c = 1; c + 3 < N; c += 4) { t0 = kc_max3(t0, v[c], v[c + 1]); t1 = kc_max3(t1, v[c + 2], v[c + 3]); }
#pragma unroll
  for (int c = (N - 1) / 4 * 4 + 1; c < N; c++) t0 = fmaxf(t0, v[c]);
  return fmaxf(t0, t1);
}
// (x, y) * (s, s) + (t, t), and sums of pairs
__device__ __forceinline__ float2 kc_fma2(float x, float y, float s, float t) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmov.b64 c, {%5, %5};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(x), "f"(y), "f"(s), "f"(t));
  return r;
}
__device__ __forceinline__ void kc_add2(float2& s, float x, float y) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}" : "+f"(s.x), "+f"(s.y) : "f"(x), "f"(y));
}
// Sixteen codes as halves times their row's scale.  int8: (1024 + 128 + code) s - 1152 s is exact in one operation, as long as 1152 s
// is a half (`small`).
template <int FMT>
__device__ __forceinline__ void kc_widen(const uint4& x, __half2 s, __half2 bias, bool small, __half2 (&h)[8]) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  if (FMT == KVQ_INT8 && small) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t lo = __byte_perm(w[i], 0x64646464u, 0x4140), hi = __byte_perm(w[i], 0x64646464u, 0x4342);
      h[2 * i] = __hfma2(*reinterpret_cast<const __half2*>(&lo), s, bias);
      h[2 * i + 1] = __hfma2(*reinterpret_cast<const __half2*>(&hi), s, bias);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    kvq_widen<FMT>(w[i], h[2 * i], h[2 * i + 1]);
    h[2 * i] = __hmul2_rn(h[2 * i], s);
    h[2 * i + 1] = __hmul2_rn(h[2 * i + 1], s);
  }
}

template <int FMT, int HD>
__global__ void __launch_bounds__(KC_THREADS, 1) kvq_chunk_kernel(const KvqChunkArgs a) {
  constexpr int KB = HD / 64;                     // 64-column blocks of a tile's rows
  constexpr uint32_t BLOCK = 128 * 128;           // bytes of a block of 128 rows
  using Cfg = KcCfg<HD>;
  extern __shared__ __align__(1024) unsigned char kc_raw[];
  unsigned char* sQ = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(kc_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* sK = sQ + 2 * Cfg::Q_BYTES;
  unsigned char* sV = sK + 2 * Cfg::KV_BYTES;
  __shared__ __align__(8) uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_low[2], p_high[2], o_full[2], q_full[2], met, plan_full[KC_PLAN], plan_empty[KC_PLAN];
  __shared__ KcPiece s_plan[KC_PLAN];
  __shared__ uint32_t s_tmem;
  __shared__ unsigned int s_ticket;
  __shared__ long long s_sum[KC_THREADS / 32], s_find[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = uniform_warp();
  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(&k_full[i], 4); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], 4); mbar_init(&v_empty[i], 1); mbar_init(&s_full[i], 1);
      mbar_init(&p_low[i], 4); mbar_init(&p_high[i], 4); mbar_init(&o_full[i], 1); mbar_init(&q_full[i], 4);
    }
    mbar_init(&met, 8);
    for (int i = 0; i < KC_PLAN; i++) { mbar_init(&plan_full[i], 1); mbar_init(&plan_empty[i], 17); }  // all warps but the plan's own and the last two
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = s_tmem;
  pdl_launch();  // only now: see tcgen05.cuh
  pdl_wait();

  // ---- the line of tiles: how long it is, and where this CTA's stretch begins.  Entry e = (sequence, item of it), all kv heads.
  const long long entries = (long long)a.B * a.max_tiles;
  auto weight = [&](long long e) -> long long {
    KcPiece p;
    if (e >= entries) return 0;
    const int b = a.max_tiles == 1 ? (int)e : (int)(e / a.max_tiles);
    return (long long)kc_item(a, b, (int)(e - (long long)b * a.max_tiles), p) * a.c.G;
  };
  const long long w_first = weight(tid);
  long long total = w_first;
  for (long long e = tid + KC_THREADS; e < entries; e += KC_THREADS) total += weight(e);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) s_sum[warp] = total;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < KC_THREADS / 32; w++) total += s_sum[w];
  const int ctas = (int)max(1ll, min((long long)gridDim.x, (total + a.grain - 1) / a.grain));
  const long long u_lo = (int)blockIdx.x < ctas ? blockIdx.x * total / ctas : 0, u_hi = (int)blockIdx.x < ctas ? (blockIdx.x + 1) * total / ctas : 0;
  long long before = 0;
  for (long long base = 0; base < entries && u_lo < u_hi; base += KC_THREADS) {  // the same for all threads
    const long long mine = base == 0 ? w_first : weight(base + tid);
    long long sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long below = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += below;
    }
    __syncthreads();
    if (lane == 31) s_sum[warp] = sum;
    __syncthreads();
    long long ahead = before;
    for (int w = 0; w < warp; w++) ahead += s_sum[w];
    if (ahead + sum - mine <= u_lo && u_lo < ahead + sum) { s_find[0] = ahead + sum - mine; s_find[1] = base + tid; }
#pragma unroll
    for (int w = 0; w < KC_THREADS / 32; w++) before += s_sum[w];
    if (before > u_lo) break;
  }
  __syncthreads();

  bool ok = true;
  uint32_t planned = 0;
  auto next = [&](KcPiece& p) -> bool {  // the next piece of the plan, for a converged warp
    const uint32_t slot = planned % KC_PLAN;
    ok = ok && mbar_wait(&plan_full[slot], (planned / KC_PLAN) & 1);
    if (!ok) return false;
    p = s_plan[slot];
    __syncwarp();
    if (lane == 0) ft_arrive(&plan_empty[slot]);
    planned++;
    return p.b >= 0;
  };
  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KC_MMA_REGS));
    if (warp == 17) {
      // ---- the plan: a walk along this CTA's stretch of the line
      long long u = u_lo, at = u_lo < u_hi ? s_find[0] : 0;  // at: first tile of (b, tile, head 0)
      int b = 0, tile = 0;
      if (u_lo < u_hi) { b = (int)(s_find[1] / a.max_tiles); tile = (int)(s_find[1] % a.max_tiles); }
      for (;; planned++) {
        const uint32_t slot = planned % KC_PLAN;
        if (planned >= KC_PLAN) ok = mbar_wait(&plan_empty[slot], (planned / KC_PLAN - 1) & 1);
        if (!ok) break;
        KcPiece p;
        p.b = -1;
        if (u < u_hi) {
          int n;
          for (;;) {
            n = kc_item(a, b, tile, p);
            if (n == 0) { tile = 0; b++; continue; }  // the items of a sequence are its first ones
            if (u < at + (long long)n * a.c.G) break;
            at += (long long)n * a.c.G;
            if (++tile == a.max_tiles) { tile = 0; b++; }
          }
          p.b = b; p.tile = tile; p.n_tiles = n;
          p.g = (int)(u - at) / n;  // both below 2^31: see the limits of the cache
          const long long item = at + (long long)p.g * n;
          p.j0 = (int)(u - item);
          p.j1 = (int)min((long long)n, u_hi - item);
          u = item + p.j1;
          p.c_lo = p.pieces = 0;
          if (p.j1 - p.j0 < n) {
            p.c_lo = (int)(((item + 1) * ctas - 1) / total);
            p.pieces = (int)(((item + n) * ctas - 1) / total) - p.c_lo + 1;
          }
        }
        if (lane == 0) { s_plan[slot] = p; ft_arrive(&plan_full[slot]); }
        if (p.b < 0) break;
      }
      if (!ok && lane == 0) atomicCAS(a.err, 0, 1);
    } else if (warp == 16) {
      // ---- products
      constexpr uint32_t id_s = (1u << 4) | ((uint32_t)(KC_KEYS >> 3) << 17) | (8u << 24);
      constexpr uint32_t id_o = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | (8u << 24);
      uint32_t tiles = 0, loaded[2] = {0, 0}, made[2] = {0, 0};  // key tiles, items and score tiles so far
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) umma_commit(bar);
      };
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && mbar_wait(bar, parity);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      };
      auto qk = [&](int q, uint32_t slot) {
        const uint64_t da = umma_desc(sQ + (size_t)q * Cfg::Q_BYTES), db = umma_desc(sK + (size_t)slot * Cfg::KV_BYTES);
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < KB; c++)
#pragma unroll
            for (int k = 0; k < 4; k++)
              umma_f16(tmem + q * 128, da + c * (BLOCK >> 4) + 2 * k, db + c * (BLOCK >> 4) + 2 * k, id_s, (c > 0 || k > 0) ? 1u : 0u);
          umma_commit(&s_full[q]);
        }
        made[q]++;
      };
      KcPiece p;
      while (next(p)) {
        const int n = p.j1 - p.j0, streams = p.n * a.n_rep - p.tile * KC_ROWS > 128 ? 2 : 1;
        for (int q = 0; q < streams; q++) wait(&q_full[q], loaded[q]++ & 1);
        wait(&k_full[tiles & 1], (tiles >> 1) & 1);
        if (!ok) break;
        for (int q = 0; q < streams; q++) qk(q, tiles & 1);
        commit(&k_empty[tiles & 1]);
        for (int j = 0; j < n && ok; j++, tiles++) {
          const uint32_t slot = tiles & 1, then = slot ^ 1;
          wait(&v_full[slot], (tiles >> 1) & 1);
          for (int q = 0; q < streams && ok; q++) {
            const uint64_t db = umma_desc_mn(sV + (size_t)slot * Cfg::KV_BYTES, BLOCK);
            wait(&p_low[q], (made[q] - 1) & 1);  // the weights of the first 64 keys, then of the others
            if (!ok) break;
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < KC_KEYS / 32; k++)  // 16 rows of values = 2048 bytes further
                umma_f16_ts(tmem + 256 + q * 128, tmem + q * 128 + k * 8, db + k * 128, id_o, (j > 0 || k > 0) ? 1u : 0u);
            }
            wait(&p_high[q], (made[q] - 1) & 1);
            if (!ok) break;
            if (elect_one()) {
#pragma unroll
              for (int k = KC_KEYS / 32; k < KC_KEYS / 16; k++)
                umma_f16_ts(tmem + 256 + q * 128, tmem + q * 128 + k * 8, db + k * 128, id_o, 1u);
              umma_commit(&o_full[q]);
            }
            if (j + 1 < n) {
              if (q == 0) wait(&k_full[then], ((tiles + 1) >> 1) & 1);
              if (ok) qk(q, then);
            }
          }
          if (!ok) break;
          commit(&v_empty[slot]);
          if (j + 1 < n) commit(&k_empty[then]);
        }
      }
      if (!ok && lane == 0) atomicCAS(a.err, 0, 2);
    }
  } else if (warp >= 8) {
    // ---- keys, or values: codes to halves, into 128-byte swizzled rows
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KC_WIDEN_REGS));
    constexpr int LPR = HD / 16, ROWS = 128 / LPR, N = 128 / ROWS;  // lanes to a row of codes; rows at a time; times
    const bool values = warp >= 12;
    const int u = tid & 127, sub = u % LPR, row = u / LPR;
    const uint8_t* codes = values ? a.c.v : a.c.k;
    const __half* scales = reinterpret_cast<const __half*>(a.c.scales) + (values ? 1 : 0);
    uint64_t* full = values ? v_full : k_full;
    uint64_t* empty = values ? v_empty : k_empty;
    unsigned char* tile = values ? sV : sK;
    // a thread's pieces of a row: columns 16 sub .. are two 16-byte pieces of a block's row.  The upper block's lanes begin with the second,
    // so that eight lanes write to eight different places of a row.
    const int c0 = (sub & 3) * 2, flip = HD == 128 ? sub >> 2 : 0;
    tile += (sub >> 2) * BLOCK + row * 128;
    const uint32_t o0 = ((c0 + flip) ^ (row & 7)) << 4, o1 = ((c0 + 1 - flip) ^ (row & 7)) << 4;  // (row + 16 i keeps row & 7)
    uint32_t tiles = 0;
    KcPiece p;
    while (next(p)) {
      const int32_t* bt = p.bt ? p.bt : a.c.block_table;  // (a slot outside the cache: some row, nobody sees it)
      const int mask = (1 << a.c.page_shift) - 1, last = max(p.T - 1, 0);
      // lane l & 7: the page of the tile's positions 16 l ..; positions past the end are the last one, masked
      auto pages_of = [&](int j) { return bt[min(j * KC_KEYS + (lane & 7) * 16, last) >> a.c.page_shift]; };
      uint4 x[N];
      __half s[N];
      auto load = [&](int j, int pages) {
#pragma unroll
        for (int i = 0; i < N; i++) {
          const int page = __shfl_sync(0xffffffffu, pages, (row + i * ROWS) >> 4);
          const uint32_t at = ((uint32_t)(page * a.c.G + p.g) << a.c.page_shift) + (uint32_t)(min(j * KC_KEYS + row + i * ROWS, last) & mask);
          x[i] = ld_stream_128(codes + (size_t)at * HD + sub * 16);
          s[i] = scales[2 * (size_t)at];
        }
      };
      int pages = pages_of(p.j0);
      load(p.j0, pages);
      if (p.j0 + 1 < p.j1) pages = pages_of(p.j0 + 1);
      for (int j = p.j0; j < p.j1; j++, tiles++) {
        const uint32_t slot = tiles & 1;
        if (tiles >= 2) ok = mbar_wait(&empty[slot], ((tiles >> 1) - 1) & 1);
        if (!ok) break;
        unsigned char* to = tile + (size_t)slot * Cfg::KV_BYTES;
        bool small = true;
#pragma unroll
        for (int i = 0; i < N; i++) small = small && !(__half2float(s[i]) > 56.f);
        small = FMT == KVQ_INT8 && __all_sync(0xffffffffu, small);
#pragma unroll
        for (int i = 0; i < N; i++) {
          const __half2 sc = __half2half2(s[i]);
          __half2 h[8];
          kc_widen<FMT>(x[i], sc, __hmul2_rn(sc, __floats2half2_rn(-1152.f, -1152.f)), small, h);
          const uint4 lo = *reinterpret_cast<const uint4*>(h), hi = *reinterpret_cast<const uint4*>(h + 4);
          *reinterpret_cast<uint4*>(to + i * ROWS * 128 + o0) = flip ? hi : lo;
          *reinterpret_cast<uint4*>(to + i * ROWS * 128 + o1) = flip ? lo : hi;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) ft_arrive(&full[slot]);
        if (j + 1 < p.j1) load(j + 1, pages);
        if (j + 2 < p.j1) pages = pages_of(j + 2);
      }
    }
    if (!ok && lane == 0) atomicCAS(a.err, 0, 1);
  } else {
    // ---- softmax: a thread for each row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(KC_SOFT_REGS));
    const int q = warp >> 2, r = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), S = lanes + q * 128, O = lanes + 256 + q * 128;
    unsigned char* rows_at = sQ + (size_t)q * Cfg::Q_BYTES + (warp & 3) * 32 * 128;  // this warp's 32 rows of queries, and of results behind them
    uint32_t made = 0, meetings = 0;  // score tiles so far, and times that the two streams have met
    auto meet = [&]() {  // of all softmax warps, with a limit: bar.sync would wait for a warp that gave up
      __syncwarp();
      if (lane == 0) ft_arrive(&met);
      ok = mbar_wait(&met, meetings++ & 1) && ok;
    };
    KcPiece p;
    while (next(p)) {
      const int n = p.j1 - p.j0, rows = p.n * a.n_rep - p.tile * KC_ROWS, mine = q * 128 + r;  // rows of the item, and this thread's
      const bool active = rows > q * 128;  // the stream has rows at all
      const int i = (p.tile * KC_ROWS + mine) / a.n_rep, h = p.tile * KC_ROWS + mine - i * a.n_rep;
      const long long row = (long long)(a.first ? a.first[p.b] : p.b) + (long long)i * a.step, pos = (long long)p.p0 + i;
      const bool there = mine < rows && row >= 0 && row < a.R;
      const bool outside = p.bt == nullptr || pos < 0 || pos >= a.c.max_ctx;
      const int lim = !there ? p.T - 1 : (int)max(-1ll, min(pos, (long long)p.T - 1));  // last key that the row sees
      const int head = p.g * a.n_rep + h;
      float m = -INFINITY;
      float2 l = make_float2(0.f, 0.f);
      if (active) {
        // the warp's 32 rows, HD / 8 lanes to a row
        const long long from = there ? row * a.ldq + head * HD : -1;
        constexpr int W = HD / 8, PER = 32 / W;
#pragma unroll
        for (int k = 0; k < 32; k += PER * 8) {
          uint4 x[8];
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const long long at = __shfl_sync(0xffffffffu, from, k + e * PER + lane / W);
            x[e] = at < 0 ? make_uint4(0, 0, 0, 0) : ld_128(a.q + at + lane % W * 8);
          }
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const int rr = k + e * PER + lane / W, c = lane % W;
            *reinterpret_cast<uint4*>(rows_at + (c >> 3) * BLOCK + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = x[e];
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) ft_arrive(&q_full[q]);
        for (int j = 0; j < n; j++, made++) {
          ok = mbar_wait(&s_full[q], made & 1);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          // the first 64 scores stay in registers, the others are read twice
          float v[64], y[32];
          tmem_ld32(S, v);
          tmem_ld32(S + 32, v + 32);
          kc_landed<64>(v);
          tmem_ld32(S + 64, y);
          const int key = (p.j0 + j) * KC_KEYS;
          const bool all = __all_sync(0xffffffffu, key + KC_KEYS - 1 <= lim);
          auto hide = [&](float* x, int k, int count) {
            if (all) return;
#pragma unroll
            for (int c = 0; c < count; c++) x[c] = k + c <= lim ? x[c] : -INFINITY;
          };
          hide(v, key, 64);
          float top = kc_max<64>(-INFINITY, v);
          kc_landed<32>(y);
          {
            float z[32];
            tmem_ld32(S + 96, z);
            hide(y, key + 64, 32);
            top = kc_max<32>(top, y);
            kc_landed<32>(z);
            hide(z, key + 96, 32);
            top = kc_max<32>(top, z);
          }
          top *= a.scale2;
          if (__any_sync(0xffffffffu, top > m + 8.f)) {
            const float then = fmaxf(m, top), fade = then == m ? 1.f : ft_ex2(m - then);
            m = then;
            l.x *= fade;
            l.y *= fade;
            if (j > 0) {
              ok = mbar_wait(&o_full[q], (made - 1) & 1);  // the product before has to be in O
              if (!ok) break;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
              for (int c = 0; c < HD; c += 32) {
                uint32_t w[32];
                tmem_ld32(O + c, y);
                kc_landed<32>(y);
#pragma unroll
                for (int k = 0; k < 32; k++) w[k] = __float_as_uint(y[k] * fade);
                tmem_st32(O + c, w);
              }
            }
          }
          const float base = m == -INFINITY ? 0.f : -m, sc = a.scale2;
          auto weights = [&](const float* x, uint32_t* w, int count) {
#pragma unroll
            for (int k = 0; k < count; k += 2) {
              const float2 e = kc_fma2(x[k], x[k + 1], sc, base);
              const float e0 = ft_ex2(e.x), e1 = ft_ex2(e.y);
              kc_add2(l, e0, e1);
              asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[k / 2]) : "f"(e1), "f"(e0));
            }
          };
          auto ready = [&](uint64_t* bar) {
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) ft_arrive(bar);
          };
          uint32_t w[32];
          weights(v, w, 64);
          tmem_st32(S, w);
          tmem_ld32(S + 64, v);
          tmem_ld32(S + 96, v + 32);
          ready(&p_low[q]);
          kc_landed<64>(v);
          hide(v, key + 64, 64);
          weights(v, w, 64);
          tmem_st32(S + 32, w);
          ready(&p_high[q]);
        }
        if (ok) {
          ok = mbar_wait(&o_full[q], (made - 1) & 1);
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
      }
      // ---- the result, or a piece of it
      const bool whole = n == p.n_tiles;
      float* part = a.part + (size_t)(2 * blockIdx.x + (p.j0 == 0 ? 1 : 0)) * kc_part_floats(HD);  // [hd / 4][256][4], maxima, sums
      const long long to = there ? row * a.ldo + head * HD : -1;
      // 32 columns from c on of the warp's rows, as halves in the place of its queries (whose products are done)
      auto gather = [&](int c, const float* o, float f) {
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const __half2 x = __floats2half2_rn(o[k + 2 * e] * f, o[k + 2 * e + 1] * f);
            w[e] = outside ? 0u : *reinterpret_cast<const uint32_t*>(&x);
          }
          const int g = (c + k) / 8;
          *reinterpret_cast<uint4*>(rows_at + (g >> 3) * BLOCK + lane * 128 + (((g & 7) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      };
      auto store = [&]() {  // and out, HD / 8 lanes to a row
        __syncwarp();
        constexpr int W = HD / 8, PER = 32 / W;
#pragma unroll 4
        for (int k = 0; k < 32; k += PER) {
          const int rr = k + lane / W, c = lane % W;
          const long long at = __shfl_sync(0xffffffffu, to, rr);
          const uint4 x = *reinterpret_cast<const uint4*>(rows_at + (c >> 3) * BLOCK + rr * 128 + (((c & 7) ^ (rr & 7)) << 4));
          if (at >= 0) *reinterpret_cast<uint4*>(a.out + at + c * 8) = x;
        }
        __syncwarp();
      };
      const float sum_here = l.x + l.y;
      if (active && ok) {
        const float f = sum_here == 0.f ? 0.f : __fdiv_rn(1.f, sum_here);
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          float o[32];
          tmem_ld32(O + c, o);
          kc_landed<32>(o);
          if (whole) {
            gather(c, o, f);
          } else {
#pragma unroll
            for (int k = 0; k < 32; k += 4) __stcg(reinterpret_cast<float4*>(part) + (size_t)((c + k) / 4) * KC_ROWS + mine, make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
          }
        }
        if (whole) store();
        else { __stcg(part + HD * KC_ROWS + mine, m); __stcg(part + HD * KC_ROWS + KC_ROWS + mine, sum_here); }
      }
      if (whole) continue;
      // ---- an item that CTAs c_lo .. share: the last to arrive adds its pieces up in this order
      __threadfence();
      meet();
      if (tid == 0) {
        s_ticket = atomicAdd(&a.tickets[p.c_lo], 1u);
        if (s_ticket == (unsigned)(p.pieces - 1)) a.tickets[p.c_lo] = 0;
      }
      meet();
      const bool last = s_ticket == (unsigned)(p.pieces - 1);
      meet();  // read by all before the next item's
      if (!last || !active || !ok) continue;
      __threadfence();
      auto piece = [&](int k) -> const float* { return a.part + (size_t)(2 * (p.c_lo + k) + (k == 0 ? 1 : 0)) * kc_part_floats(HD); };
      float top = -INFINITY, sum = 0.f;
#pragma unroll 4
      for (int k = 0; k < p.pieces; k++) top = fmaxf(top, __ldcg(piece(k) + HD * KC_ROWS + mine));
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 4
      for (int k = 0; k < p.pieces; k++)
        sum = fmaf(__ldcg(piece(k) + HD * KC_ROWS + KC_ROWS + mine), ft_ex2(__ldcg(piece(k) + HD * KC_ROWS + mine) - base), sum);
      const float f = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        float o[32];
#pragma unroll
        for (int k = 0; k < 32; k++) o[k] = 0.f;
#pragma unroll 2
        for (int k = 0; k < p.pieces; k++) {
          const float w = ft_ex2(__ldcg(piece(k) + HD * KC_ROWS + mine) - base);
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float4 y = __ldcg(reinterpret_cast<const float4*>(piece(k)) + (size_t)(c / 4 + e) * KC_ROWS + mine);
            o[4 * e] = fmaf(y.x, w, o[4 * e]); o[4 * e + 1] = fmaf(y.y, w, o[4 * e + 1]);
            o[4 * e + 2] = fmaf(y.z, w, o[4 * e + 2]); o[4 * e + 3] = fmaf(y.w, w, o[4 * e + 3]);
          }
        }
        gather(c, o, f);
      }
      store();
    }
    if (!ok && lane == 0) atomicCAS(a.err, 0, 3);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 16) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

template <int FMT, int HD>
static int launch_chunk(jg_dev* dev, const KvqChunkArgs& a) {
  auto kern = kvq_chunk_kernel<FMT, HD>;
  static bool ready[8] = {};
  if (!ready[dev->ordinal & 7]) {
    cudaFuncAttributes f;
    JG_CUDA(cudaFuncGetAttributes(&f, kern));
    if (f.numRegs < KC_REGS) {  // the warpgroups' shares are cut out of what the CTA is launched with: a smaller launch would wait for registers for ever
      jg_set_error("kvq_attn: the kernel was compiled for %d registers a thread, and wants %d", f.numRegs, KC_REGS);
      return JG_ENOTSUP;
    }
    JG_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)KcCfg<HD>::SMEM));
    ready[dev->ordinal & 7] = true;
  }
  dev->tc_pending = true;
  return jg_launch(dev, "kvq_attn", kern, dim3((unsigned)kc_ctas(dev)), dim3(KC_THREADS), KcCfg<HD>::SMEM, a);
}

int kvq_chunk(jg_dev* dev, int format, int hd, const KvqChunkArgs& a) {
  if (format == JG_KVQ_INT8) return hd == 64 ? launch_chunk<KVQ_INT8, 64>(dev, a) : launch_chunk<KVQ_INT8, 128>(dev, a);
  return hd == 64 ? launch_chunk<KVQ_E4M3, 64>(dev, a) : launch_chunk<KVQ_E4M3, 128>(dev, a);
}
