// Attention of chunks over the 8-bit KV cache on the 5th-generation tensor cores (jg_kvq_attn beyond a few queries).
//
// One pass over the keys with a running maximum: S = Q.K^T, P = 2^(S - m), O += P.V, l += sum P; O / l at the end.  The codes of a tile
// of keys and values become halves, code * scale exactly, on their way into the shared-memory tiles that the products read, so
// a tile crosses HBM as bytes and no 16-bit copy of the cache exists.
//
// A query row is a (position, query head) of one kv head; an item is 256 rows, two streams of 128, over the keys that its last
// row sees, in tiles of 128.  Four warpgroups: 0 and 1 softmax, a stream each, a thread per row; 2 loads and widens K and V; the first
// warp of 3 issues the products.  While one stream's exponentials run, the other's products do.  Tensor memory: S of both streams (P
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

constexpr int KC_THREADS = 512, KC_REGS = 128;                                // at launch
constexpr int KC_SOFT_REGS = 184, KC_WIDEN_REGS = 104, KC_MMA_REGS = 40;      // 2 * 184 + 104 + 40 = 4 * 128
static_assert(2 * KC_SOFT_REGS + KC_WIDEN_REGS + KC_MMA_REGS <= 4 * KC_REGS, "register shares exceed what a CTA is launched with");

template <int HD>
struct KcCfg {
  static constexpr uint32_t Q_BYTES = 128 * HD * 2, KV_BYTES = KC_KEYS * HD * 2;
  static constexpr size_t SMEM = 2 * Q_BYTES + 4 * KV_BYTES + 1024;
};

// One piece of work: the tiles [j0, j1) of an item.
struct KcPiece {
  int b, tile, g, j0, j1, n_tiles;  // n_tiles: of the whole item
  long long item;                   // its first tile on the line
  int p0, n, T;                     // first new position and number of new positions of the sequence; keys that the item looks at
  const int32_t* bt;                // null: the slot lies outside the cache
};

// What a sequence is, and how many key tiles item `tile` of it has (0: no such item).
__device__ __forceinline__ int kc_item(const KvqChunkArgs& a, int b, int tile, KcPiece& p) {
  const int sq = a.seq ? a.seq[b] : b;
  p.n = max(0, a.count ? min(a.count[b], a.max_count) : a.max_count);
  if ((long long)tile * KC_ROWS >= (long long)p.n * a.n_rep) return 0;
  p.p0 = a.pos[b];
  const bool have = (unsigned)sq < (unsigned)a.c.n_seq;
  p.bt = have ? a.c.block_table + (size_t)sq * a.c.max_pages : nullptr;
  const long long last = min((long long)p.n, ((long long)(tile + 1) * KC_ROWS - 1) / a.n_rep + 1);  // positions up to the item's end
  p.T = have ? (int)max(0ll, min((long long)p.p0 + last, (long long)a.c.max_ctx)) : 0;
  return max(1, (p.T + KC_KEYS - 1) / KC_KEYS);
}

// Walks a CTA's stretch [u, u_hi) of the line, all lanes of a warp alike.
struct KcWalk {
  long long u, u_hi, at;  // at: first tile of (b, tile, head 0)
  int b, tile;
  __device__ __forceinline__ bool next(const KvqChunkArgs& a, KcPiece& p) {
    if (u >= u_hi) return false;
    int n;
    for (;;) {
      n = kc_item(a, b, tile, p);
      if (n == 0) { tile = 0; b++; continue; }  // the items of a sequence are its first ones
      if (u < at + (long long)n * a.c.G) break;
      at += (long long)n * a.c.G;
      if (++tile == a.max_tiles) { tile = 0; b++; }
    }
    p.b = b; p.tile = tile; p.n_tiles = n;
    p.g = (int)((u - at) / n);
    p.item = at + (long long)p.g * n;
    p.j0 = (int)(u - p.item);
    p.j1 = (int)min((long long)n, u_hi - p.item);
    u = p.item + p.j1;
    return true;
  }
};

template <int FMT, int HD>
__global__ void __launch_bounds__(KC_THREADS, 1) kvq_chunk_kernel(const KvqChunkArgs a) {
  constexpr int KB = HD / 64;                     // 64-column blocks of a tile's rows
  constexpr uint32_t BLOCK = 128 * 128;           // bytes of a block of 128 rows
  using Cfg = KcCfg<HD>;
  extern __shared__ __align__(1024) unsigned char kc_raw[];
  unsigned char* sQ = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(kc_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* sK = sQ + 2 * Cfg::Q_BYTES;
  unsigned char* sV = sK + 2 * Cfg::KV_BYTES;
  __shared__ __align__(8) uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], q_full[2], met;
  __shared__ uint32_t s_tmem;
  __shared__ unsigned int s_ticket;
  __shared__ long long s_sum[KC_THREADS / 32], s_find[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = uniform_warp();
  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(&k_full[i], 4); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], 4); mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&o_full[i], 1); mbar_init(&q_full[i], 4);
    }
    mbar_init(&met, 8);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 12) {
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
    return e < entries ? (long long)kc_item(a, (int)(e / a.max_tiles), (int)(e % a.max_tiles), p) * a.c.G : 0;
  };
  long long total = 0;
  for (long long e = tid; e < entries; e += KC_THREADS) total += weight(e);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) s_sum[warp] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < KC_THREADS / 32; w++) total += s_sum[w];
  const long long ctas = max(1ll, min((long long)gridDim.x, (total + a.grain - 1) / a.grain));
  KcWalk walk;
  walk.u = blockIdx.x < ctas ? blockIdx.x * total / ctas : 0;
  walk.u_hi = blockIdx.x < ctas ? (blockIdx.x + 1) * total / ctas : 0;
  long long before = 0;
  for (long long base = 0; base < entries && walk.u < walk.u_hi; base += KC_THREADS) {  // the same for all threads
    const long long mine = weight(base + tid);
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
    if (ahead + sum - mine <= walk.u && walk.u < ahead + sum) { s_find[0] = ahead + sum - mine; s_find[1] = base + tid; }
    for (int w = 0; w < KC_THREADS / 32; w++) before += s_sum[w];
    if (before > walk.u) break;
  }
  __syncthreads();
  if (walk.u < walk.u_hi) { walk.at = s_find[0]; walk.b = (int)(s_find[1] / a.max_tiles); walk.tile = (int)(s_find[1] % a.max_tiles); }

  KcPiece p;
  bool ok = true;
  if (warp >= 12) {
    // ---- products
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KC_MMA_REGS));
    if (warp == 12) {
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
      while (ok && walk.next(a, p)) {
        const int n = p.j1 - p.j0, streams = (long long)p.n * a.n_rep - (long long)p.tile * KC_ROWS > 128 ? 2 : 1;
        for (int q = 0; q < streams; q++) wait(&q_full[q], loaded[q]++ & 1);
        wait(&k_full[tiles & 1], (tiles >> 1) & 1);
        if (!ok) break;
        for (int q = 0; q < streams; q++) qk(q, tiles & 1);
        commit(&k_empty[tiles & 1]);
        for (int j = 0; j < n && ok; j++, tiles++) {
          const uint32_t slot = tiles & 1, then = slot ^ 1;
          wait(&v_full[slot], (tiles >> 1) & 1);
          for (int q = 0; q < streams && ok; q++) {
            wait(&p_full[q], (made[q] - 1) & 1);
            if (!ok) break;
            const uint64_t db = umma_desc_mn(sV + (size_t)slot * Cfg::KV_BYTES, BLOCK);
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < KC_KEYS / 16; k++)  // 16 rows of values = 2048 bytes further
                umma_f16_ts(tmem + 256 + q * 128, tmem + q * 128 + k * 8, db + k * 128, id_o, (j > 0 || k > 0) ? 1u : 0u);
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
    // ---- keys and values: codes to halves, into 128-byte swizzled rows
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KC_WIDEN_REGS));
    constexpr int LPR = HD / 16, ROWS = 128 / LPR, N = 128 / ROWS;  // lanes to a row of codes; rows at a time; times
    const int u = tid - 256, sub = u % LPR, row = u / LPR;
    uint32_t tiles = 0;
    while (ok && walk.next(a, p)) {
      uint4 kc[N], vc[N];
      __half2 sc[N], next[N];
      uint32_t at[N];  // rows of the pool
      const int32_t* bt = p.bt ? p.bt : a.c.block_table;  // (a slot outside the cache: some row, nobody sees it)
      auto where = [&](int j) {
#pragma unroll
        for (int i = 0; i < N; i++) at[i] = (uint32_t)kvq_row(a.c, bt, max(0, min(j * KC_KEYS + row + i * ROWS, p.T - 1)), p.g);  // past the end: the last row, masked
      };
      auto load_k = [&]() {
#pragma unroll
        for (int i = 0; i < N; i++) { kc[i] = ld_128(a.c.k + (size_t)at[i] * HD + sub * 16); next[i] = a.c.scales[at[i]]; }
      };
      auto load_v = [&]() {
#pragma unroll
        for (int i = 0; i < N; i++) vc[i] = ld_128(a.c.v + (size_t)at[i] * HD + sub * 16);
      };
      auto widen = [&](const uint4& x, __half2 s, unsigned char* tile, int rw) {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
        __half2 h[8];
#pragma unroll
        for (int i = 0; i < 4; i++) kvq_widen<FMT>(w[i], h[2 * i], h[2 * i + 1]);
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = __hmul2_rn(h[i], s);
        // columns 16 sub ..: two 16-byte pieces of a block's row; the upper block's lanes begin with the second, so that eight lanes
        // write to eight different places of a row
        unsigned char* to = tile + (sub >> 2) * BLOCK + rw * 128;
        const int c0 = (sub & 3) * 2, flip = HD == 128 ? sub >> 2 : 0;
        const uint4 lo = *reinterpret_cast<const uint4*>(h), hi = *reinterpret_cast<const uint4*>(h + 4);
        *reinterpret_cast<uint4*>(to + (((c0 + flip) ^ (rw & 7)) << 4)) = flip ? hi : lo;
        *reinterpret_cast<uint4*>(to + (((c0 + 1 - flip) ^ (rw & 7)) << 4)) = flip ? lo : hi;
      };
      auto done = [&](uint64_t* bar) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) ft_arrive(bar);
      };
      where(p.j0);
      load_k();
      load_v();
      for (int j = p.j0; j < p.j1 && ok; j++, tiles++) {
        const uint32_t slot = tiles & 1;
        if (tiles >= 2) ok = mbar_wait(&k_empty[slot], ((tiles >> 1) - 1) & 1);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < N; i++) { sc[i] = next[i]; widen(kc[i], __low2half2(sc[i]), sK + (size_t)slot * Cfg::KV_BYTES, row + i * ROWS); }
        done(&k_full[slot]);
        if (j + 1 < p.j1) { where(j + 1); load_k(); }
        if (tiles >= 2) ok = mbar_wait(&v_empty[slot], ((tiles >> 1) - 1) & 1);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < N; i++) widen(vc[i], __high2half2(sc[i]), sV + (size_t)slot * Cfg::KV_BYTES, row + i * ROWS);
        done(&v_full[slot]);
        if (j + 1 < p.j1) load_v();
      }
    }
    if (!ok && lane == 0) atomicCAS(a.err, 0, 1);
  } else {
    // ---- softmax: a thread for each row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(KC_SOFT_REGS));
    const int q = warp >> 2, r = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), S = lanes + q * 128, O = lanes + 256 + q * 128;
    uint32_t made = 0, meetings = 0;  // score tiles so far, and times that the two streams have met
    auto meet = [&]() {  // of all softmax warps, with a limit: bar.sync would wait for a warp that gave up
      __syncwarp();
      if (lane == 0) ft_arrive(&met);
      ok = mbar_wait(&met, meetings++ & 1) && ok;
    };
    while (ok && walk.next(a, p)) {
      const int n = p.j1 - p.j0;
      const long long rows = (long long)p.n * a.n_rep, mine = (long long)p.tile * KC_ROWS + q * 128 + r;
      const bool active = rows - (long long)p.tile * KC_ROWS > q * 128;  // the stream has rows at all
      const int i = (int)(mine / a.n_rep), h = (int)(mine - (long long)i * a.n_rep);
      const long long row = (long long)(a.first ? a.first[p.b] : p.b) + (long long)i * a.step, pos = (long long)p.p0 + i;
      const bool there = mine < rows && row >= 0 && row < a.R;
      const bool outside = p.bt == nullptr || pos < 0 || pos >= a.c.max_ctx;
      const int lim = !there ? p.T - 1 : (int)max(-1ll, min(pos, (long long)p.T - 1));  // last key that the row sees
      __half* out = a.out + (size_t)(there ? row : 0) * a.ldo + (size_t)(p.g * a.n_rep + h) * HD;
      float m = -INFINITY, l = 0.f;
      if (active) {
        const __half* x = a.q + (size_t)(there ? row : 0) * a.ldq + (size_t)(p.g * a.n_rep + h) * HD;
        unsigned char* to = sQ + (size_t)q * Cfg::Q_BYTES + r * 128;
#pragma unroll
        for (int c = 0; c < HD / 8; c++)
          *reinterpret_cast<uint4*>(to + (c >> 3) * BLOCK + (((c & 7) ^ (r & 7)) << 4)) = there ? ld_128(x + c * 8) : make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) ft_arrive(&q_full[q]);
        float v[KC_KEYS];
        for (int j = 0; j < n; j++, made++) {
          ok = mbar_wait(&s_full[q], made & 1);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
          for (int c = 0; c < KC_KEYS; c += 32) tmem_ld32(S + c, v + c);
          tmem_ld_wait();
          const int key = (p.j0 + j) * KC_KEYS;
          if (!__all_sync(0xffffffffu, key + KC_KEYS - 1 <= lim)) {
#pragma unroll
            for (int c = 0; c < KC_KEYS; c++) v[c] = key + c <= lim ? v[c] : -INFINITY;
          }
          float t0 = v[0], t1 = v[1], t2 = v[2], t3 = v[3];
#pragma unroll
          for (int c = 4; c < KC_KEYS; c += 4) { t0 = fmaxf(t0, v[c]); t1 = fmaxf(t1, v[c + 1]); t2 = fmaxf(t2, v[c + 2]); t3 = fmaxf(t3, v[c + 3]); }
          const float top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3)) * a.scale2;
          if (__any_sync(0xffffffffu, top > m + 8.f)) {
            const float then = fmaxf(m, top), fade = then == m ? 1.f : ft_ex2(m - then);
            m = then;
            l *= fade;
            if (j > 0) {
              ok = mbar_wait(&o_full[q], (made - 1) & 1);  // the product before has to be in O
              if (!ok) break;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
              for (int c = 0; c < HD; c += 32) {
                float o[32];
                uint32_t w[32];
                tmem_ld32(O + c, o);
                tmem_ld_wait();
#pragma unroll
                for (int k = 0; k < 32; k++) w[k] = __float_as_uint(o[k] * fade);
                tmem_st32(O + c, w);
              }
            }
          }
          const float base = m == -INFINITY ? 0.f : m, sc = a.scale2;
          float a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
#pragma unroll
          for (int c = 0; c < KC_KEYS; c += 64) {
            uint32_t w[32];
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              const float x0 = ft_ex2(fmaf(v[c + 2 * k], sc, -base)), x1 = ft_ex2(fmaf(v[c + 2 * k + 1], sc, -base));
              const float x2 = ft_ex2(fmaf(v[c + 2 * k + 2], sc, -base)), x3 = ft_ex2(fmaf(v[c + 2 * k + 3], sc, -base));
              a0 += x0; a1 += x1; a2 += x2; a3 += x3;
              asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[k]) : "f"(x1), "f"(x0));
              asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[k + 1]) : "f"(x3), "f"(x2));
            }
            tmem_st32(S + c / 2, w);
          }
          l += (a0 + a1) + (a2 + a3);
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) ft_arrive(&p_full[q]);
        }
        if (ok) {
          ok = mbar_wait(&o_full[q], (made - 1) & 1);
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
      }
      // ---- the result, or a piece of it
      auto store = [&](int c, const float* o, float f) {  // eight values of the row
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const __half2 x = __floats2half2_rn(o[2 * k] * f, o[2 * k + 1] * f);
          w[k] = outside ? 0u : *reinterpret_cast<const uint32_t*>(&x);
        }
        *reinterpret_cast<uint4*>(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
      };
      const bool whole = n == p.n_tiles;
      float* part = a.part + (size_t)(2 * blockIdx.x + (p.j0 == 0 ? 1 : 0)) * kc_part_floats(HD) + q * 128 + r;  // [hd / 4][256][4], maxima, sums
      if (active && ok) {
        const float f = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          float o[32];
          tmem_ld32(O + c, o);
          tmem_ld_wait();
          if (whole) {
            if (there)
#pragma unroll
              for (int k = 0; k < 32; k += 8) store(c + k, o + k, f);
          } else {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              __stcg(reinterpret_cast<float4*>(part - (q * 128 + r)) + (size_t)((c + k) / 4) * KC_ROWS + q * 128 + r, make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
          }
        }
        if (!whole) { __stcg(part + HD * KC_ROWS, m); __stcg(part + HD * KC_ROWS + KC_ROWS, l); }
      }
      if (whole) continue;
      // ---- an item that CTAs c_lo .. c_hi share: the last to arrive adds its pieces up in this order
      const int c_lo = (int)(((p.item + 1) * ctas - 1) / total), pieces = (int)(((p.item + p.n_tiles) * ctas - 1) / total) - c_lo + 1;
      __threadfence();
      meet();
      if (tid == 0) {
        s_ticket = atomicAdd(&a.tickets[c_lo], 1u);
        if (s_ticket == (unsigned)(pieces - 1)) a.tickets[c_lo] = 0;
      }
      meet();
      const bool last = s_ticket == (unsigned)(pieces - 1);
      meet();  // read by all before the next item's
      if (!last || !active || !ok) continue;
      __threadfence();
      auto piece = [&](int k) -> const float* { return a.part + (size_t)(2 * (c_lo + k) + (k == 0 ? 1 : 0)) * kc_part_floats(HD); };
      float top = -INFINITY, sum = 0.f;
      for (int k = 0; k < pieces; k++) top = fmaxf(top, __ldcg(piece(k) + HD * KC_ROWS + q * 128 + r));
      const float base = top == -INFINITY ? 0.f : top;
      for (int k = 0; k < pieces; k++)
        sum = fmaf(__ldcg(piece(k) + HD * KC_ROWS + KC_ROWS + q * 128 + r), ft_ex2(__ldcg(piece(k) + HD * KC_ROWS + q * 128 + r) - base), sum);
      const float f = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        float o[32];
#pragma unroll
        for (int k = 0; k < 32; k++) o[k] = 0.f;
        for (int k = 0; k < pieces; k++) {
          const float w = ft_ex2(__ldcg(piece(k) + HD * KC_ROWS + q * 128 + r) - base);
#pragma unroll
          for (int x = 0; x < 8; x++) {
            const float4 y = __ldcg(reinterpret_cast<const float4*>(piece(k)) + (size_t)(c / 4 + x) * KC_ROWS + q * 128 + r);
            o[4 * x] = fmaf(y.x, w, o[4 * x]); o[4 * x + 1] = fmaf(y.y, w, o[4 * x + 1]);
            o[4 * x + 2] = fmaf(y.z, w, o[4 * x + 2]); o[4 * x + 3] = fmaf(y.w, w, o[4 * x + 3]);
          }
        }
        if (there)
#pragma unroll
          for (int k = 0; k < 32; k += 8) store(c + k, o + k, f);
      }
    }
    if (!ok && lane == 0) atomicCAS(a.err, 0, 3);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 12) {
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
    if (f.numRegs != KC_REGS) {  // the warpgroups' shares are cut out of what the CTA is launched with: a smaller launch would wait for registers for ever
      jg_set_error("kvq_attn: the kernel was compiled for %d registers a thread, not %d", f.numRegs, KC_REGS);
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
