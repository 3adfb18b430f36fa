// Attention of chunks over the 8-bit KV cache on the 5th-generation tensor cores (jg_kvq_attn beyond a few queries).
//
// One pass over the keys with a running maximum: S = Q.K^T, P = 2^(S - m), O += P.V, l += sum P; O / l at the end.  The codes of a tile
// of keys and values become halves, code * scale exactly, on their way into the shared-memory tiles that the products read, so
// a tile crosses HBM as bytes and no 16-bit copy of the cache exists.
//
// A query row is a (position, query head) of one kv head; an item is 256 rows, two streams of 128, over the keys that its last
// row sees, in tiles of 128; an item of up to 128 rows has its tiles take turns between the streams, whose outputs meet at its end.  Five
// warpgroups: softmax of either stream, a thread per row; one that loads and widens K, one for V; the last issues the products and keeps
// the plan.  While one stream's exponentials run, the other's products do; a product with V begins when the first half of its weights is
// there.  Tensor memory: S of both streams (P takes its place as 16-bit pairs), O of both.  A row's maximum is a reference that its scores
// may pass by 2^8 before O is rescaled in tensor memory, which is rare behind the first tiles.
//
// The tiles of all items are one line, cut evenly over one CTA for each SM.  An item that several CTAs share meets in a workspace: two
// pieces are added up by the last CTA to arrive (3 to 4 us), more by all of its CTAs, a share of the rows each; always in their order.  These wait for
// one another, so the launch is a cooperative one, which begins behind its predecessor: 2 us a call more than the times of the comparisons below,
// which were taken with launches that begin early.
//
// What bounds it: per 256 rows x 128 keys x 128 columns four products of 512 cycles at the tensor peak, and 32768 exponentials at 16 a
// cycle, 2048 cycles either way; such a unit takes 4000.  2048 positions of the 8B behind 6001, fp8: 239 us, 0.98 PFLOP/s, in
// a short run, 265 us, 0.89 PFLOP/s, in a long one under the power limit (1.66 GHz).  The tensor pipe
// and the exponentials' are each busy 47 % of the time, issue slots 45 %: the two softmax warps of a scheduler wait for tensor memory, their
// maxima and votes, and fill each other's gaps only in part (of 233 us: without exponentials 200, without a softmax 171, without widening 212).
// Tried and slower: two threads to a row on 16 warps (290: registers), the widening on 16 warps (265), products of half a tile's keys, all 128
// scores in registers, a share of the exponentials as polynomials; rows of 64 values with weights apart from the scores, so that the next
// scores are made meanwhile (82.3 and 83.9 us for 24 ragged chunks of the 1B).
#include <math.h>

#include "flash_tc.cuh"
#include "kvquant.cuh"
#include "kvquant_chunk.cuh"

// Warps 0-3 and 4-7 softmax, 8-11 keys, 12-15 values, 16 products, 17 plan; 18 and 19 fill up the last warpgroup.
constexpr int KC_THREADS = 640, KC_REGS = 96;                                 // registers at launch
constexpr int KC_SOFT_REGS = 144, KC_WIDEN_REGS = 72, KC_MMA_REGS = 48;       // and from then on, by warpgroup
static_assert(2 * KC_SOFT_REGS + 2 * KC_WIDEN_REGS + KC_MMA_REGS <= 5 * KC_REGS, "register shares exceed what a CTA is launched with");
constexpr int KC_PLAN = 4;  // pieces that the plan is ahead
constexpr int KC_FEW = 2, KC_BATCH = 4;  // pieces that one CTA adds up; pieces whose loads are in flight together
constexpr int KC_HALF = KC_KEYS / 2;  // keys of a step of the softmax

template <int HD>
struct KcCfg {
  static constexpr uint32_t Q_BYTES = 128 * HD * 2, KV_BYTES = KC_KEYS * HD * 2;
  static constexpr size_t SMEM = 2 * Q_BYTES + 4 * KV_BYTES + 1024;
};

// A piece of work: the key tiles [j0, j1) of an item.
struct KcPiece {
  const int32_t* bt;       // null: the slot lies outside the cache
  int b, g, j0, j1;        // b < 0: no more pieces
  int row0;                // the item's first row of the sequence's
  int left;                // its rows; up to 128: its key tiles take turns between the two streams
  int n_tiles;             // of the whole item
  int p0, n, T;            // first new position and number of new positions of the sequence; keys that the item looks at
  int c_lo, pieces;        // the CTAs that share the item
};

// What a sequence is, and how many key tiles item `tile` of it has (0: no such item).
__device__ __forceinline__ int kc_item(const KvqChunkArgs& a, int b, int tile, int rows, KcPiece& p) {
  p.row0 = tile * rows;
  const int sq = a.seq ? a.seq[b] : b, count = a.count ? a.count[b] : a.max_count;
  p.p0 = a.pos[b];
  p.n = max(0, min(count, a.max_count));
  const int first = a.first ? a.first[b] : b;
  if ((long long)first + (long long)(p.n - 1) * a.step >= a.R) p.n = first < a.R ? (int)(((long long)a.R - 1 - first) / a.step) + 1 : 0;  // rows there are
  if ((long long)tile * rows >= (long long)p.n * a.n_rep) return 0;
  p.left = min(rows, p.n * a.n_rep - p.row0);
  const bool have = (unsigned)sq < (unsigned)a.c.n_seq;
  p.bt = have ? a.c.block_table + (size_t)sq * a.c.max_pages : nullptr;
  const int last = min(p.n, ((tile + 1) * rows - 1) / a.n_rep + 1);  // positions up to the item's end
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
__device__ __forceinline__ float kc_max64(const float* v) {  // in four chains
  float t0 = v[0], t1 = v[1], t2 = v[2], t3 = v[3];
#pragma unroll
  for (int c = 4; c + 8 <= 60; c += 8) {
    t0 = kc_max3(t0, v[c], v[c + 1]);
    t1 = kc_max3(t1, v[c + 2], v[c + 3]);
    t2 = kc_max3(t2, v[c + 4], v[c + 5]);
    t3 = kc_max3(t3, v[c + 6], v[c + 7]);
  }
  t0 = kc_max3(t0, v[60], v[61]);
  t1 = kc_max3(t1, v[62], v[63]);
  return fmaxf(kc_max3(t0, t1, t2), t3);
}
// Until as many CTAs have left their pieces: for a converged warp, with a limit.  They all run or have run: the launch is a cooperative one, and
// none of its CTAs waits for anything outside it.
__device__ __forceinline__ bool kc_arrived(const unsigned int* ticket, unsigned int pieces) {
  for (uint32_t i = 0; i < TC_SPIN_LIMIT; i++) {
    unsigned int n;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(ticket) : "memory");
    if (__all_sync(0xffffffffu, n >= pieces)) return true;
  }
  return false;
}
// pairs of floats: packed operands stay in register pairs, made once where they do not change
__device__ __forceinline__ uint64_t kc_pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 kc_split(uint64_t p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ uint64_t kc_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t kc_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
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
  __shared__ __align__(8) uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2][2], o_full[2][2], q_full[2], met;
  __shared__ __align__(8) uint64_t plan_full[KC_PLAN], plan_empty[KC_PLAN];
  __shared__ KcPiece s_plan[KC_PLAN];
  __shared__ uint32_t s_tmem;
  __shared__ KcPiece s_shared[2];
  __shared__ unsigned int s_ticket;
  __shared__ float2 s_ml[2][128];
  __shared__ long long s_sum[KC_THREADS / 32], s_at;
  __shared__ int s_longest[KC_THREADS / 32], s_entry;
  const int tid = threadIdx.x, lane = tid & 31, warp = uniform_warp();
  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(&k_full[i], 4); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], 4); mbar_init(&v_empty[i], 1); mbar_init(&s_full[i], 1); mbar_init(&q_full[i], 4);
      for (int half = 0; half < 2; half++) { mbar_init(&p_full[i][half], 4); mbar_init(&o_full[i][half], 1); }  // [stream][half of a key tile]
    }
    mbar_init(&met, 8);
    for (int i = 0; i < KC_PLAN; i++) { mbar_init(&plan_full[i], 1); mbar_init(&plan_empty[i], 17); }  // all warps but the plan's own and the last two
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  const uint32_t tmem = ft_columns(&s_tmem, warp == 16);

  // ---- the line of tiles: how long it is, and where this CTA's stretch begins.  Entry e = (sequence, item of it), all kv heads.  Up to 32
  // entries are the plan's own business; more are looked at by all threads.
  const int entries = a.B * a.max_tiles;
  auto tiles_of = [&](int e) -> int {
    KcPiece p;
    return e < entries ? kc_item(a, e / a.max_tiles, e % a.max_tiles, KC_ROWS, p) : 0;
  };
  auto cost = [&](int n) { return n > 0 ? (long long)(n + KC_FIXED) * a.c.G : 0ll; };
  auto warp_sum64 = [&](long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  auto scan64 = [&](long long v) {  // of this lane and those below it
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long below = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += below;
    }
    return v;
  };
  // An item costs what KC_FIXED tiles do beside its own.  Cutting one costs its CTAs a trip through memory each, 2 to 4 us: short items are
  // not cut, others not into less than KC_GRAIN tiles (45 new positions of the 8B behind 3000: 2, 3, 4, 6 tiles 20, 21, 21, 30 us).  `uncut`: none is
  // longer than KC_WHOLE tiles, or KC_SINGLE where there is a CTA for each (a prompt of 900, 8 tiles: cut 37 us, 26; of 1100, 9 tiles and 144
  // items: 42, 30; 160 items of 10 tiles: 48, 55; 8 items of 10: 20, 23; of 16: 18, 33).
  long long total = 0, u_lo = 0, u_hi = 0;
  int longest = 0, ctas = 1;
  bool uncut = false;
  auto share = [&]() {
    const long long most = uncut ? total : total / KC_GRAIN;
    ctas = (int)max(1ll, min((long long)gridDim.x, most));
    if ((int)blockIdx.x >= ctas) return;
    u_lo = kvq_cut<KC_BITS>(total, ctas, blockIdx.x);  // 512 CTAs at most: see the launch
    u_hi = kvq_cut<KC_BITS>(total, ctas, blockIdx.x + 1);
  };
  if (entries > 32) {
    for (int e = tid; e < entries; e += KC_THREADS) {
      const int n = tiles_of(e);
      total += cost(n);
      longest = max(longest, n);
    }
    total = warp_sum64(total);
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 0) { s_sum[warp] = total; s_longest[warp] = longest; }
    __syncthreads();
    total = 0;
    for (int w = 0; w < KC_THREADS / 32; w++) { total += s_sum[w]; longest = max(longest, s_longest[w]); }
    uncut = longest <= KC_WHOLE;
    share();
    long long before = 0;
    for (int base = 0; base < entries && u_lo < u_hi; base += KC_THREADS) {  // the same for all threads
      const long long mine = cost(tiles_of(base + tid)), sum = scan64(mine);
      __syncthreads();
      if (lane == 31) s_sum[warp] = sum;
      __syncthreads();
      long long ahead = before;
      for (int w = 0; w < KC_THREADS / 32; w++) { ahead += w < warp ? s_sum[w] : 0; before += s_sum[w]; }
      if (ahead + sum - mine <= u_lo && u_lo < ahead + sum) { s_at = ahead + sum - mine; s_entry = base + tid; }
      if (before > u_lo) break;
    }
    __syncthreads();
  }

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
      long long at;  // first tile of (b, tile, head 0)
      int entry, rows = KC_ROWS, per = a.max_tiles;  // of an item; items of a sequence
      bool single = false;
      if (entries > 32) {
        at = s_at;
        entry = s_entry;
      } else {
        int items;
        long long mine, sum;
        auto look = [&]() {  // at items of this many rows
          KcPiece p;
          const int n = lane < a.B * per ? kc_item(a, lane / per, lane % per, rows, p) : 0;
          longest = __reduce_max_sync(0xffffffffu, n);
          items = __popc(__ballot_sync(0xffffffffu, n > 0)) * a.c.G;
          uncut = longest <= (items <= (int)gridDim.x ? KC_SINGLE : KC_WHOLE);
          single = uncut && items <= (int)gridDim.x;
          mine = single ? (n > 0 ? a.c.G : 0) : cost(n);
          sum = scan64(mine);
          total = __shfl_sync(0xffffffffu, sum, 31);
        };
        look();
        // Items that leave half of the CTAs idle become items of half the rows, whose two streams share their keys (512 new positions of the
        // 8B 16.6 us, 18.7 without); and where each CTA has one at most, they count alike (18.7 us, 19.3 without).
        if (entries <= 16 && 2 * (uncut ? items : total / KC_GRAIN) <= (long long)gridDim.x) {
          rows = KC_ROWS / 2;
          per *= 2;
          look();
        }
        share();
        entry = max(0, __ffs(__ballot_sync(0xffffffffu, sum > u_lo)) - 1);
        at = __shfl_sync(0xffffffffu, sum - mine, entry);
      }
      long long u = u_lo;
      int b = entry / per, tile = entry % per;
      for (;; planned++) {
        const uint32_t slot = planned % KC_PLAN;
        if (planned >= KC_PLAN) ok = mbar_wait(&plan_empty[slot], (planned / KC_PLAN - 1) & 1);
        if (!ok) break;
        KcPiece p;
        p.b = -1;
        while (u < u_hi) {
          const int n = kc_item(a, b, tile, rows, p);
          if (n == 0) { tile = 0; b++; continue; }  // the items of a sequence are its first ones
          const int span = single ? 1 : n + KC_FIXED;  // of an item on the line; its tiles are behind its fixed cost
          if (u >= at + (long long)span * a.c.G) {
            at += (long long)span * a.c.G;
            if (++tile == per) { tile = 0; b++; }
            continue;
          }
          p.g = (int)(u - at) / span;  // both below 2^31: see the limits of the cache
          const long long item = at + (long long)p.g * span;
          if (uncut) {  // the CTA in whose stretch it begins has all of it
            const bool mine = u == item;
            u = item + span;
            if (!mine) continue;
            p.j0 = 0;
            p.j1 = n;
          } else {
            p.j0 = max(0, (int)(u - item) - KC_FIXED);
            u = min(item + span, u_hi);
            p.j1 = max(0, (int)(u - item) - KC_FIXED);
            if (p.j0 == p.j1) continue;
          }
          p.b = b; p.n_tiles = n;
          p.c_lo = p.pieces = 0;
          if (p.j1 - p.j0 < n) {
            const long long begin = item + KC_FIXED;
            p.c_lo = kvq_owner(total, ctas, begin);
            p.pieces = kvq_owner(total, ctas, begin + n - 1) - p.c_lo + 1;
          }
          break;
        }
        if (lane == 0) { s_plan[slot] = p; ft_arrive(&plan_full[slot]); }
        if (p.b < 0) break;
      }
      if (!ok && lane == 0) atomicCAS(a.err, 0, JG_WAIT_KVQ_PLAN);
    } else if (warp == 16) {
      // ---- products
      constexpr uint32_t id_s = (1u << 4) | ((uint32_t)(KC_KEYS >> 3) << 17) | (8u << 24);
      constexpr uint32_t id_o = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | (8u << 24);
      uint32_t tiles = 0, loaded[2] = {0, 0}, made[2] = {0, 0};  // key tiles, items, and key tiles of either stream so far
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) umma_commit(bar);
      };
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && mbar_wait(bar, parity);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      };
      auto qk = [&](int q, uint32_t slot, int rows) {  // scores of a stream: of which 128 rows, over which tile of keys
        const uint64_t da = umma_desc(sQ + (size_t)rows * Cfg::Q_BYTES), db = umma_desc(sK + (size_t)slot * Cfg::KV_BYTES);
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < KB; c++)
#pragma unroll
            for (int k = 0; k < 4; k++)
              umma_f16(tmem + q * 128, da + c * (BLOCK >> 4) + 2 * k, db + c * (BLOCK >> 4) + 2 * k, id_s, (c > 0 || k > 0) ? 1u : 0u);
          umma_commit(&s_full[q]);
        }
      };
      auto pv = [&](int q, uint32_t slot, bool first) {  // its weights times a tile of values, half a tile at a time
        const uint64_t db = umma_desc_mn(sV + (size_t)slot * Cfg::KV_BYTES, BLOCK);
#pragma unroll
        for (int half = 0; half < 2; half++) {
          wait(&p_full[q][half], made[q] & 1);
          if (ok && elect_one()) {
#pragma unroll
            for (int k = half * (KC_HALF / 16); k < (half + 1) * (KC_HALF / 16); k++)  // 16 rows of values = 2048 bytes further
              umma_f16_ts(tmem + 256 + q * 128, tmem + q * 128 + k * 8, db + k * 128, id_o, (!first || k > 0) ? 1u : 0u);
            umma_commit(&o_full[q][half]);
          }
        }
        made[q]++;
      };
      KcPiece p;
      while (next(p)) {
        const int n = p.j1 - p.j0;
        if (p.left <= 128) {
          wait(&q_full[0], loaded[0]++ & 1);
          auto scores = [&](int j) {  // of tile j, for the stream whose turn it is
            const uint32_t slot = (tiles + j) & 1;
            wait(&k_full[slot], ((tiles + j) >> 1) & 1);
            if (ok) qk(j & 1, slot, 0);
            if (ok) commit(&k_empty[slot]);
          };
          for (int j = 0; j < 2 && j < n; j++) scores(j);
          for (int j = 0; j < n && ok; j++) {
            const uint32_t slot = (tiles + j) & 1;
            wait(&v_full[slot], ((tiles + j) >> 1) & 1);
            if (ok) pv(j & 1, slot, j < 2);
            if (ok) commit(&v_empty[slot]);
            if (j + 2 < n) scores(j + 2);
          }
          tiles += n;
          continue;
        }
        for (int q = 0; q < 2; q++) wait(&q_full[q], loaded[q]++ & 1);
        wait(&k_full[tiles & 1], (tiles >> 1) & 1);
        if (!ok) break;
        for (int q = 0; q < 2; q++) qk(q, tiles & 1, q);
        commit(&k_empty[tiles & 1]);
        for (int j = 0; j < n && ok; j++, tiles++) {
          const uint32_t slot = tiles & 1, then = slot ^ 1;
          const bool more = j + 1 < n;
          wait(&v_full[slot], (tiles >> 1) & 1);
          for (int q = 0; q < 2 && ok; q++) {
            pv(q, slot, j == 0);
            if (more && q == 0) wait(&k_full[then], ((tiles + 1) >> 1) & 1);
            if (more && ok) qk(q, then, q);
          }
          if (!ok) break;
          commit(&v_empty[slot]);
          if (more) commit(&k_empty[then]);
        }
      }
      if (!ok && lane == 0) atomicCAS(a.err, 0, JG_WAIT_KVQ_PRODUCTS);
    }
  } else if (warp >= 8) {
    // ---- keys, or values: codes to halves, into 128-byte swizzled rows
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KC_WIDEN_REGS));
    // Four lanes take a 64-column block of a row, lanes 4-7 the row behind it: in 128-byte swizzled rows the eight 16-byte pieces that they
    // write at a time fall on different banks.  A warp has PER neighbouring rows of each of the N groups of ROWS.
    constexpr int ROWS = HD == 128 ? 16 : 32, N = 128 / ROWS, PER = ROWS / 4;
    const bool values = warp >= 12;
    const int u = tid & 127, sub = HD == 128 ? (u & 3) + ((u >> 3) & 1) * 4 : u & 3, row = HD == 128 ? (u >> 4) * 2 + ((u >> 2) & 1) : u >> 2;
    const uint8_t* codes = (values ? a.c.v : a.c.k) + sub * 16;
    const __half* scales = reinterpret_cast<const __half*>(a.c.scales) + (values ? 1 : 0);
    uint64_t* full = values ? v_full : k_full;
    uint64_t* empty = values ? v_empty : k_empty;
    unsigned char* tile = (values ? sV : sK) + (sub >> 2) * BLOCK + row * 128;
    const uint32_t o0 = (((sub & 3) * 2) ^ (row & 7)) << 4, o1 = (((sub & 3) * 2 + 1) ^ (row & 7)) << 4;  // (row + i * ROWS keeps row & 7)
    uint32_t tiles = 0;
    KcPiece p;
    while (next(p)) {
      const int32_t* bt = p.bt ? p.bt : a.c.block_table;  // (a slot outside the cache: some row, nobody sees it)
      const int mask = (1 << a.c.page_shift) - 1, last = max(p.T - 1, 0);
      // Lane l & 7 looks after positions 16 (l & 7) .. of a tile, which lie in one page: its page, and the row of the pool where they begin.
      // Positions past the end are the last one, masked.
      auto page_of = [&](int j) { return bt[min(j * KC_KEYS + (lane & 7) * 16, last) >> a.c.page_shift]; };
      auto first_row = [&](int j, int page) { return ((uint32_t)(page * a.c.G + p.g) << a.c.page_shift) + (uint32_t)(min(j * KC_KEYS + (lane & 7) * 16, last) & mask); };
      // A piece of a row is asked for as soon as the one of the tile before it is done with, so that all have a tile's time to come.
      uint4 x[N];
      uint32_t begin = 0;  // of the tile whose rows are asked for: first_row
      int room = 0;        // its rows up to the last position
      auto row_at = [&](int r) {  // row of the pool of the tile's row r
        const uint32_t b0 = __shfl_sync(0xffffffffu, begin, r >> 4);
        return b0 + (uint32_t)(room >= KC_KEYS - 1 ? r & 15 : max(0, min(r & 15, room - (r & ~15))));
      };
      auto tile_at = [&](int j, int page) { begin = first_row(j, page); room = last - j * KC_KEYS; };
      auto scale_at = [&]() {  // lane l: the scale of row (l / PER) * ROWS + l % PER of the warp's rows
        return __half2float(scales[2 * (size_t)row_at((lane / PER % N) * ROWS + (warp & 3) * PER + lane % PER)]);
      };
      auto codes_at = [&](int i) { return ld_stream_128(codes + (size_t)row_at(row + i * ROWS) * HD); };
      int page = page_of(p.j0), page2 = page_of(p.j0 + 1);
      tile_at(p.j0, page);
      float s = scale_at();
#pragma unroll
      for (int i = 0; i < N; i++) x[i] = codes_at(i);
      page = page2;
      page2 = page_of(p.j0 + 2);
      for (int j = p.j0; j < p.j1; j++, tiles++) {
        const uint32_t slot = tiles & 1;
        if (tiles >= 2) ok = mbar_wait(&empty[slot], ((tiles >> 1) - 1) & 1);
        if (!ok) break;
        unsigned char* to = tile + (size_t)slot * Cfg::KV_BYTES;
        const bool small = FMT == KVQ_INT8 && __all_sync(0xffffffffu, !(s > 56.f)), more = j + 1 < p.j1;
        float then = 0.f;
        if (more) {
          tile_at(j + 1, page);
          then = scale_at();
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
          const __half2 sc = __float2half2_rn(__shfl_sync(0xffffffffu, s, i * PER + (row & (PER - 1))));
          __half2 h[8];
          kc_widen<FMT>(x[i], sc, __hmul2_rn(sc, __floats2half2_rn(-1152.f, -1152.f)), small, h);
          if (more) x[i] = codes_at(i);
          *reinterpret_cast<uint4*>(to + i * ROWS * 128 + o0) = *reinterpret_cast<const uint4*>(h);
          *reinterpret_cast<uint4*>(to + i * ROWS * 128 + o1) = *reinterpret_cast<const uint4*>(h + 4);
        }
        s = then;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) ft_arrive(&full[slot]);
        page = page2;
        page2 = page_of(j + 3);
      }
    }
    if (!ok && lane == 0) atomicCAS(a.err, 0, JG_WAIT_KVQ_CODES);
  } else {
    // ---- softmax: a thread for each row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(KC_SOFT_REGS));
    const int q = warp >> 2, r = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), S = lanes + q * 128, O = lanes + 256 + q * 128;
    unsigned char* rows_at = sQ + (size_t)q * Cfg::Q_BYTES + (warp & 3) * 32 * 128;  // this warp's 32 rows of queries, and of results behind them
    const uint64_t scale2 = kc_pair(a.scale2, a.scale2);
    uint32_t made = 0, meetings = 0, turn = 0;  // score tiles so far, times that the two streams have met, split items
    auto meet = [&]() {  // of all softmax warps, with a limit: bar.sync would wait for a warp that gave up
      __syncwarp();
      if (lane == 0) ft_arrive(&met);
      ok = mbar_wait(&met, meetings++ & 1) && ok;
    };
    // What this thread's row is, worked out from the plan where it is needed: the loop over tiles has no registers to keep it in.
    auto mine_of = [&](const KcPiece& p) { return p.left <= 128 ? r : q * 128 + r; };  // of the item's rows
    auto row_of = [&](const KcPiece& p, int& head, int& i) -> long long {  // row of queries and results, or -1
      const int at = p.row0 + mine_of(p);
      i = at / a.n_rep;
      head = p.g * a.n_rep + at - i * a.n_rep;
      const long long row = (long long)(a.first ? a.first[p.b] : p.b) + (long long)i * a.step;
      return at < p.n * a.n_rep && row >= 0 && row < a.R ? row : -1;
    };
    int shared = 0;  // pieces of items that other CTAs have pieces of
    for (;; planned++) {
      const uint32_t planned_slot = planned % KC_PLAN;
      ok = ok && mbar_wait(&plan_full[planned_slot], (planned / KC_PLAN) & 1);
      if (!ok) break;
      const KcPiece& p = s_plan[planned_slot];
      if (p.b < 0) break;
      auto release = [&]() {
        __syncwarp();
        if (lane == 0) ft_arrive(&plan_empty[planned_slot]);
      };
      const bool split = p.left <= 128, idle = p.left <= mine_of(p) - lane;  // this warp has no rows
      const int n = split ? (p.j1 - p.j0 + 1 - q) / 2 : p.j1 - p.j0;  // tiles of this stream
      int lim;  // last key that the row sees
      float m = -INFINITY;
      uint64_t l0 = kc_pair(0.f, 0.f), l1 = l0;  // the sum, in four parts
      {
        int head, i;
        const long long row = row_of(p, head, i);
        lim = row < 0 ? p.T - 1 : (int)max(-1ll, min((long long)p.p0 + i, (long long)p.T - 1));
        if (!split || q == 0) {
          const long long from = row < 0 ? -1 : row * a.ldq + head * HD;
          // the warp's 32 rows, HD / 8 lanes to a row
          constexpr int W = HD / 8, PER = 32 / W;
#pragma unroll 4
          for (int k = 0; k < 32; k += PER) {
            const int rr = k + lane / W, c = lane % W;
            const long long at = __shfl_sync(0xffffffffu, from, rr);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                         ::"r"(smem_u32(rows_at + (c >> 3) * BLOCK + rr * 128 + (((c & 7) ^ (rr & 7)) << 4))), "l"(a.q + max(at, 0ll) + c * 8), "r"(at < 0 ? 0 : 16)
                         : "memory");  // zeros for rows that there are not
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) ft_arrive(&q_full[q]);
        }
      }
      int key = (p.j0 + (split ? q : 0)) * KC_KEYS;
      for (int j = 0; j < n; j++, made++, key += split ? 2 * KC_KEYS : KC_KEYS) {
        ok = mbar_wait(&s_full[q], made & 1);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (idle) {  // whatever lies in the place of its weights concerns rows that nobody stores
          if (lane == 0) { ft_arrive(&p_full[q][0]); ft_arrive(&p_full[q][1]); }
          continue;
        }
        // Two halves of 64 keys, each a step of its own of the running maximum: the first one's product with V runs while the second is here.
        const bool all = __all_sync(0xffffffffu, key + KC_KEYS - 1 <= lim);
        float v[64];
        tmem_ld32(S, v);
        tmem_ld32(S + 32, v + 32);
#pragma unroll
        for (int half = 0; half < 2; half++) {
          kc_landed<64>(v);
          if (!all) {
#pragma unroll
            for (int c = 0; c < 64; c++) v[c] = key + half * 64 + c <= lim ? v[c] : -INFINITY;
          }
          const float top = kc_max64(v) * a.scale2;
          if (__any_sync(0xffffffffu, top > m + 8.f)) {
            const float then = fmaxf(m, top), fade = then == m ? 1.f : ex2(m - then);
            m = then;
            const uint64_t f2 = kc_pair(fade, fade);
            l0 = kc_fma2(l0, f2, kc_pair(0.f, 0.f));
            l1 = kc_fma2(l1, f2, kc_pair(0.f, 0.f));
            if (j > 0 || half > 0) {  // the product before has to be in O
              ok = half == 0 ? mbar_wait(&o_full[q][1], (made - 1) & 1) : mbar_wait(&o_full[q][0], made & 1);
              if (!ok) break;
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
              for (int c = 0; c < HD; c += 32) {
                float y[32];
                uint32_t w[32];
                tmem_ld32(O + c, y);
                kc_landed<32>(y);
#pragma unroll
                for (int k = 0; k < 32; k++) w[k] = __float_as_uint(y[k] * fade);
                tmem_st32(O + c, w);
              }
            }
          }
          const float base = m == -INFINITY ? 0.f : -m;
          const uint64_t base2 = kc_pair(base, base);
          uint32_t w[32];
#pragma unroll
          for (int k = 0; k < 64; k += 4) {
            const float2 x = kc_split(kc_fma2(kc_pair(v[k], v[k + 1]), scale2, base2)), y = kc_split(kc_fma2(kc_pair(v[k + 2], v[k + 3]), scale2, base2));
            const float x0 = ex2(x.x), x1 = ex2(x.y), y0 = ex2(y.x), y1 = ex2(y.y);
            l0 = kc_add2(l0, kc_pair(x0, x1));
            l1 = kc_add2(l1, kc_pair(y0, y1));
            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[k / 2]) : "f"(x1), "f"(x0));
            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[k / 2 + 1]) : "f"(y1), "f"(y0));
          }
          tmem_st32(S + half * 32, w);
          if (half == 0) {
            tmem_ld32(S + 64, v);
            tmem_ld32(S + 96, v + 32);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) ft_arrive(&p_full[q][half]);
        }
        if (!ok) break;
      }
      if (ok && n > 0) {
        ok = mbar_wait(&o_full[q][1], (made - 1) & 1);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      }
      const float2 la = kc_split(l0), lb = kc_split(l1);
      float sum = (la.x + la.y) + (lb.x + lb.y), own = 1.f, others = 0.f;  // the shares of the two streams' outputs
      // ---- the streams of a split item: a row's two outputs lie in the same lane of tensor memory
      if (split && p.n_tiles > 1) {
        float2* ml = s_ml[turn++ & 1] + r;  // two in turn: a stream without tiles would be ahead of the other
        if (q == 1) *ml = make_float2(m, sum);
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        meet();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (q == 0) {
          const float2 o = *ml;
          const float then = fmaxf(m, o.x), base = then == -INFINITY ? 0.f : then;
          own = ex2(m - base);
          others = ex2(o.x - base);
          sum = sum * own + o.y * others;
          m = then;
        }
      }
      const bool both = split && p.j1 - p.j0 > 1, absent = split && q == 1;  // the other stream has outputs; this one's are the other's to store
      auto outputs = [&](int c, float* o) {  // 32 columns of the row
        tmem_ld32(O + c, o);
        kc_landed<32>(o);
        if (!both) return;
        float x[32];
        tmem_ld32(O + 128 + c, x);
        kc_landed<32>(x);
#pragma unroll
        for (int k = 0; k < 32; k++) o[k] = o[k] * own + x[k] * others;
      };
      // ---- the result, or a piece of it
      const bool whole = p.j1 - p.j0 == p.n_tiles;
      float* part = a.part + (size_t)kvq_slot(blockIdx.x, p.j0 == 0) * kc_part_floats(HD);  // [hd / 4][256][4], maxima, sums
      int head, i;
      const long long row = row_of(p, head, i), to = row < 0 ? -1 : row * a.ldo + head * HD;
      const bool outside = p.bt == nullptr || (long long)p.p0 + i < 0 || (long long)p.p0 + i >= a.c.max_ctx;
      // 32 columns from c on of the warp's rows, as halves in the place of its queries (whose products are done).  Zeros where there is nothing to see;
      // where all scores are -inf (an infinite query) the sum is 0 and the row NaN, as a softmax is.
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
      const int at = q * 128 + r;
      if (ok && !idle && !absent) {
        const float f = __fdiv_rn(1.f, sum);
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          float o[32];
          outputs(c, o);
          if (whole) {
            gather(c, o, f);
          } else {
#pragma unroll
            for (int k = 0; k < 32; k += 4) __stcg(reinterpret_cast<float4*>(part) + (size_t)((c + k) / 4) * KC_ROWS + at, make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
          }
        }
        if (whole) {
          store();
        } else {
          __stcg(part + HD * KC_ROWS + at, m);
          __stcg(part + HD * KC_ROWS + KC_ROWS + at, sum);
        }
      }
      if (whole) { release(); continue; }
      // ---- a piece of an item that CTAs c_lo .. share.  Two pieces are added up by the last CTA to arrive; of more every CTA adds up its share
      // behind all its own work, or one would read them all (2048 positions behind 6001, two pieces: 231 us, 237 with shares; 45 behind
      // 1900, three: 28, 24; behind 16000, 18: 72, 41).
      const bool few = p.pieces <= KC_FEW;
      if (!few && tid == 0) s_shared[shared] = p;
      meet();
      if (!few) {
        if (tid == 0) {
          __threadfence();  // all warps' pieces, which this thread knows of by their meeting, ahead of the count
          atomicAdd(&a.tickets[kc_ticket(p.c_lo)], 1u);
        }
        shared++;
        release();
        continue;
      }
      if (tid == 0) {
        __threadfence();
        s_ticket = atomicAdd(&a.tickets[kc_ticket(p.c_lo)], 1u);
        if (s_ticket == (unsigned)(p.pieces - 1)) a.tickets[kc_ticket(p.c_lo)] = 0;
        __threadfence();
      }
      meet();
      if (s_ticket != (unsigned)(p.pieces - 1) || idle || absent || !ok) { release(); continue; }
      auto piece = [&](int k) -> const float* { return a.part + (size_t)kvq_slot(p.c_lo + k, k == 0) * kc_part_floats(HD); };
      float top = -INFINITY;
#pragma unroll 4
      for (int k = 0; k < p.pieces; k++) top = fmaxf(top, __ldcg(piece(k) + HD * KC_ROWS + at));
      const float base = top == -INFINITY ? 0.f : top;
      sum = 0.f;
#pragma unroll 4
      for (int k = 0; k < p.pieces; k++) sum = fmaf(__ldcg(piece(k) + HD * KC_ROWS + KC_ROWS + at), ex2(__ldcg(piece(k) + HD * KC_ROWS + at) - base), sum);
      const float f = __fdiv_rn(1.f, sum);
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        float o[32];
#pragma unroll
        for (int k = 0; k < 32; k++) o[k] = 0.f;
#pragma unroll 1
        for (int k = 0; k < p.pieces; k++) {
          const float4* from = reinterpret_cast<const float4*>(piece(k)) + (size_t)(c / 4) * KC_ROWS + at;
          float4 y[8];
#pragma unroll
          for (int e = 0; e < 8; e++) y[e] = __ldcg(from + (size_t)e * KC_ROWS);
          const float w = ex2(__ldcg(piece(k) + HD * KC_ROWS + at) - base);
#pragma unroll
          for (int e = 0; e < 8; e++) {
            o[4 * e] = fmaf(y[e].x, w, o[4 * e]); o[4 * e + 1] = fmaf(y[e].y, w, o[4 * e + 1]);
            o[4 * e + 2] = fmaf(y[e].z, w, o[4 * e + 2]); o[4 * e + 3] = fmaf(y[e].w, w, o[4 * e + 3]);
          }
        }
        gather(c, o, f);
      }
      store();
      release();
    }
    // ---- shared items, two at most: each CTA adds up its share of the rows, a thread sixteen values at a time, pieces in their order
    for (int k = 0; k < shared && ok; k++) {
      const KcPiece& p = s_shared[k];
      unsigned int *arrived = a.tickets + kc_ticket(p.c_lo), *done = a.tickets + kc_done_ticket(gridDim.x, p.c_lo);
      ok = kc_arrived(arrived, (unsigned)p.pieces);
      if (!ok && lane == 0) atomicCAS(a.err, 0, JG_WAIT_KVQ_PIECES);
      meet();
      if (!ok) break;
      if (tid == 0 && atomicAdd(done, 1u) == (unsigned)(p.pieces - 1)) { *arrived = 0; *done = 0; }
      const int units = p.left * (HD / 16), mine = (int)blockIdx.x - p.c_lo, hi = (int)((long long)units * (mine + 1) / p.pieces);
      for (int u = (int)((long long)units * mine / p.pieces) + tid; u < hi; u += 256) {
        const int c = u / p.left, at = u - c * p.left;
        float top = -INFINITY, sum = 0.f, x[16];
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = 0.f;
#pragma unroll 1
        for (int from = 0; from < p.pieces; from += KC_BATCH) {
          float4 y[KC_BATCH][4];
          float pm[KC_BATCH], pl[KC_BATCH];
#pragma unroll
          for (int e = 0; e < KC_BATCH; e++) {
            const int n = from + e;
            if (n >= p.pieces) break;
            const float* src = a.part + (size_t)kvq_slot(p.c_lo + n, n == 0) * kc_part_floats(HD);
            pm[e] = __ldcg(src + HD * KC_ROWS + at);
            pl[e] = __ldcg(src + HD * KC_ROWS + KC_ROWS + at);
#pragma unroll
            for (int j = 0; j < 4; j++) y[e][j] = __ldcg(reinterpret_cast<const float4*>(src) + (size_t)(c * 4 + j) * KC_ROWS + at);
          }
#pragma unroll
          for (int e = 0; e < KC_BATCH; e++) {
            if (from + e >= p.pieces) break;
            const float then = fmaxf(top, pm[e]), base = then == -INFINITY ? 0.f : then, fade = ex2(top - base), f = ex2(pm[e] - base);
            top = then;
            sum = sum * fade + pl[e] * f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
              x[4 * j] = x[4 * j] * fade + y[e][j].x * f;
              x[4 * j + 1] = x[4 * j + 1] * fade + y[e][j].y * f;
              x[4 * j + 2] = x[4 * j + 2] * fade + y[e][j].z * f;
              x[4 * j + 3] = x[4 * j + 3] * fade + y[e][j].w * f;
            }
          }
        }
        const int row_head = p.row0 + at, i = row_head / a.n_rep;
        const long long row = (long long)(a.first ? a.first[p.b] : p.b) + (long long)i * a.step;
        if (row < 0 || row >= a.R) continue;
        const bool outside = p.bt == nullptr || (long long)p.p0 + i < 0 || (long long)p.p0 + i >= a.c.max_ctx;
        const float f = __fdiv_rn(1.f, sum);
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const __half2 h = __floats2half2_rn(x[2 * j] * f, x[2 * j + 1] * f);
          w[j] = outside ? 0u : *reinterpret_cast<const uint32_t*>(&h);
        }
        uint4* to = reinterpret_cast<uint4*>(a.out + row * a.ldo + (size_t)(p.g * a.n_rep + row_head - i * a.n_rep) * HD + c * 16);
        to[0] = make_uint4(w[0], w[1], w[2], w[3]);
        to[1] = make_uint4(w[4], w[5], w[6], w[7]);
      }
    }
    if (!ok && lane == 0) atomicCAS(a.err, 0, JG_WAIT_KVQ_SOFTMAX);
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
  return jg_launch_together(dev, "kvq_attn", kern, dim3((unsigned)kc_ctas(dev)), dim3(KC_THREADS), KcCfg<HD>::SMEM, a);
}

int kvq_chunk(jg_dev* dev, int format, int hd, const KvqChunkArgs& a) {
  if (format == JG_KVQ_INT8) return hd == 64 ? launch_chunk<KVQ_INT8, 64>(dev, a) : launch_chunk<KVQ_INT8, 128>(dev, a);
  return hd == 64 ? launch_chunk<KVQ_E4M3, 64>(dev, a) : launch_chunk<KVQ_E4M3, 128>(dev, a);
}
