// Attention of few queries over the 8-bit cache, bound by reading it: one new token a row, or short chunks.
//
// Queries of a (sequence, kv head) are columns, (position, query head) pairs, up to 8 * NT.  A warp takes 16 positions at a time:
//   scores^T [16 positions x columns] = K [16 x hd] . q^T        weights in 16 bits, turned by movmatrix
//   out^T [hd x columns] += V^T [hd x 16 positions] . w^T        mma.sync.m16n8k16, 32-bit sums
// The inner index of a product and the order of its rows are free as long as both operands agree, so a lane's fragments are 16
// neighbouring codes of a row: of K as they lie, of V two rows at a time with their bytes interleaved.  So a lane loads just what it
// multiplies, 16 bytes at a time and a tile ahead, straight into registers (32 sequences of 4100 positions of the 8B, with a call that
// reads the new rows back, 67 us; staged in shared memory 81).  V is multiplied by its scale as it is widened (exact), K's scale goes to
// the finished scores.  The queries' fragments lie in shared memory, each lane's own, which leaves the registers to outputs and tiles (20
// columns behind 8 x 3001 positions in L2 26.3 us, 29.5 with them in registers; from HBM 28.6.  One column group 67.5, 68.2).
//
// The running maximum is a reference that scores may pass by 2^6 before sums and outputs are rescaled: a vote a tile instead of three
// rounds of shuffles.
//
// The positions of all (sequence, kv head)s are one line of units of 16 * KS_WARPS, with some more for what each costs by itself, cut
// evenly over the CTAs: long and short conversations of a batch cost what they hold.  A CTA's stretch holds pieces of several (sequence,
// kv head)s; those that others share are left in a workspace (at most two a CTA: its first and its last), and the last to arrive puts them
// together in order.
//
// What bounds it.  32 x 4100 positions, 274 MB: 64 us, 4.3 TB/s as a whole.  The loops run at about 6 TB/s; 4.5 us pass before them
// (positions, page, first tiles: three trips through memory), 5 behind (the warps meet, the pieces), and a stretch with two pieces ends
// 4 us after one with one.  Three column groups run on eight warps an SM, 255 registers each: there latency bounds the loops (3.1 TB/s,
// issue slots 38 % busy).
#pragma once
#include "kvquant.cuh"
#include "kvquant_line.h"

struct KvqSplitArgs {
  KvqLayer c;
  const __half* x;      // rows of queries; with a new token rows of wq|wk|wv
  const __half* table;  // RoPE of the new tokens, or null
  __half* out;
  const int32_t* pos;
  const int32_t* count;
  const int32_t* first;
  const int32_t* seq;
  int ldx, ldo, R, B, H, n_rep, max_count, step, limit;  // positions from `limit` on are outside
  float scale2;                                          // log2 e / sqrt(hd)
  float* part;                                           // [2 * CTAs][columns * (hd + 2)]
  unsigned int* tickets;                                 // [2 * CTAs], zero between launches
};

constexpr int KS_THREADS = 32 * KS_WARPS, KS_CTAS = 3;  // CTAs to an SM

template <int HD, int NT>
struct KsCfg {
  static constexpr int COLS = 8 * NT, KJ = HD / 64;             // 16-byte pieces of a K row that a lane holds
  static constexpr int VB = HD / 8;                             // bytes of a V row that a lane holds
  static constexpr size_t Q_BYTES = NT * KJ * 1024;             // a warp's fragments of q
  static constexpr size_t MERGE = KS_WARPS * COLS * HD * 4;     // the warps' outputs when they meet, in the place of these
  static constexpr int PART = COLS * (HD + 2);                  // floats of a piece: outputs, maxima, sums
  static constexpr int FIXED = ks_fixed(NT);
};

#ifdef __CUDACC__
__device__ __forceinline__ void ks_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t ks_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void ks_put(uint32_t at, const uint4& x) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
}
__device__ __forceinline__ uint4 ks_get(uint32_t at, int turn) {  // anew in each turn of a loop: not to be kept in registers
  uint4 x;
  asm("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4]; // %5" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at), "r"(turn));
  return x;
}
__device__ __forceinline__ uint32_t ks_half2(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

template <int FMT, int HD, int NT, bool NEW>
__global__ void __launch_bounds__(KS_THREADS, NT == 1 ? KS_CTAS : 2) kvq_split_kernel(const KvqSplitArgs a) {
  using Cfg = KsCfg<HD, NT>;
  constexpr int COLS = Cfg::COLS, KJ = Cfg::KJ, VB = Cfg::VB, MT = HD / 16;
  extern __shared__ __align__(16) unsigned char ks_raw[];
  __shared__ float s_m[KS_WARPS + 1][COLS], s_l[KS_WARPS + 1][COLS];
  __shared__ __align__(16) __half s_new[2][HD];  // the new token's K and V as they are stored
  __shared__ unsigned int s_ticket;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, c = lane & 3;
  pdl_launch();
  pdl_wait();

  // positions of sequence b that queries look at in the cache (its new token, if any, comes on top), 0 where it has none
  auto sequence = [&](int b, int& p0, int& n, const int32_t*& bt) -> int {
    const int sq = a.seq ? a.seq[b] : b;
    p0 = a.pos[b];
    n = NEW ? 1 : max(0, a.count ? min(a.count[b], a.max_count) : a.max_count);
    bt = nullptr;
    if ((unsigned)sq >= (unsigned)a.c.n_seq) return 0;
    if (NEW && (unsigned)p0 >= (unsigned)a.limit) return 0;
    bt = a.c.block_table + (size_t)sq * a.c.max_pages;
    if (NEW) return p0;
    if (n == 0) return 0;
    return (int)max(0ll, min((long long)p0 + n, (long long)a.limit));
  };
  auto units = [&](int b) -> int {
    int p0, n;
    const int32_t* bt;
    return max(1, (sequence(b, p0, n, bt) + KS_UNIT - 1) / KS_UNIT);
  };
  // this CTA's stretch of the line of units, and the sequence that it begins in; every warp works it out for itself
  long long total = 0;
  for (int b = lane; b < a.B; b += 32) total += units(b) + Cfg::FIXED;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  total *= a.c.G;
  const long long ctas = min((long long)gridDim.x, total);
  if (blockIdx.x >= ctas) return;
  const long long u_lo = kvq_cut<KS_BITS>(total, ctas, blockIdx.x), u_hi = kvq_cut<KS_BITS>(total, ctas, blockIdx.x + 1);
  int b = 0;
  long long at = 0;  // first unit of (b, head 0)
  for (int base = 0;; base += 32) {
    const int n = base + lane < a.B ? units(base + lane) + Cfg::FIXED : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int below = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += below;
    }
    const unsigned past = __ballot_sync(0xffffffffu, at + (long long)sum * a.c.G > u_lo);
    if (past) {
      const int l = __ffs(past) - 1;
      b = base + l;
      at += (long long)__shfl_sync(0xffffffffu, sum - n, l) * a.c.G;
      break;
    }
    at += (long long)__shfl_sync(0xffffffffu, sum, 31) * a.c.G;
  }

  for (long long u = u_lo; u < u_hi; b++) {
    int p0, n_new;
    const int32_t* bt;
    const int T = sequence(b, p0, n_new, bt);
    const int n_units = max(1, (T + KS_UNIT - 1) / KS_UNIT), span = n_units + Cfg::FIXED;  // its units lie behind its fixed cost
    const long long row0 = NEW ? b : (a.first ? a.first[b] : b);
    const int n_cols = n_new * a.n_rep;
    for (int g = (int)((u - at) / span); g < a.c.G && u < u_hi; g++) {
      const long long item = at + (long long)g * span;
      const int j0 = max(0, (int)(u - item) - Cfg::FIXED);
      u = min(item + span, u_hi);
      const int j1 = max(0, (int)(u - item) - Cfg::FIXED);
      if (j0 == j1) continue;
      if (NEW && bt == nullptr) {  // a row outside the cache: nothing is stored, nothing seen
        for (int x = tid * 4; x < a.n_rep * HD; x += KS_THREADS * 4) *reinterpret_cast<uint2*>(a.out + (size_t)b * a.ldo + (size_t)g * a.n_rep * HD + x) = make_uint2(0u, 0u);
        continue;
      }
      const int t_lo = j0 * KS_UNIT, t_hi = min(T, j1 * KS_UNIT);
      const int n_tiles = t_hi > t_lo + warp * 16 ? (t_hi - t_lo - warp * 16 + KS_UNIT - 1) / KS_UNIT : 0;  // of this warp

      // ---- a tile: the lane's own pieces of 16 positions
      struct Tile {
        uint4 k[2][KJ];              // of rows r and r + 8
        uint32_t v[4][VB / 4];       // of rows 2c, 2c + 1, 2c + 8, 2c + 9
        __half2 s0, s1;              // scales of rows r and r + 8
        uint2 sv0, sv1;              // and of 2c, 2c + 1; 2c + 8, 2c + 9
      };
      auto pages_of = [&](int i) { return i + lane < n_tiles ? bt[(t_lo + (i + lane) * KS_UNIT + warp * 16) >> a.c.page_shift] : 0; };
      int pages = pages_of(0);  // lane l: page of the warp's tile 32 i + l
      auto row_of = [&](int i) -> size_t {  // of the pool, where tile i begins
        const int t0 = t_lo + i * KS_UNIT + warp * 16, page = __shfl_sync(0xffffffffu, pages, i & 31);
        return (((size_t)page * a.c.G + g) << a.c.page_shift) + (t0 & ((1 << a.c.page_shift) - 1));
      };
      auto load = [&](int i, Tile& t) {
        if (i > 0 && (i & 31) == 0) pages = pages_of(i);
        const size_t row = row_of(i);
        const uint8_t* k = a.c.k + (row + r) * HD + c * 16;
        const uint8_t* v = a.c.v + (row + 2 * c) * HD + r * VB;
        const __half2* s = a.c.scales + row;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int j = 0; j < KJ; j++) t.k[h][j] = ld_128(k + h * 8 * HD + j * 64);
#pragma unroll
        for (int h = 0; h < 4; h++) {
          const uint8_t* from = v + ((h >> 1) * 8 + (h & 1)) * HD;
          if (VB == 16) {
            const uint4 x = ld_128(from);
            t.v[h][0] = x.x; t.v[h][1] = x.y; t.v[h][VB / 4 - 2] = x.z; t.v[h][VB / 4 - 1] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(from);
            t.v[h][0] = x.x; t.v[h][1] = x.y;
          }
        }
        t.s0 = s[r];
        t.s1 = s[r + 8];
        t.sv0 = *reinterpret_cast<const uint2*>(s + 2 * c);
        t.sv1 = *reinterpret_cast<const uint2*>(s + 2 * c + 8);
      };
      // ---- fragments of q^T: the lane's column is nt * 8 + r.  Everything is asked for before anything is waited for.
      uint32_t q_at = (uint32_t)__cvta_generic_to_shared(ks_raw) + (uint32_t)(warp * Cfg::Q_BYTES + lane * 16);  // the lane's own, [nt][j][2] 512 bytes apart
      Tile tile;
      // The new token is an entry of its own when the warps' sums meet, made by the CTA with the end of its sequence and stored on the way.  Its
      // last warp has a tile less than the others at most times.
      const bool entry = NEW && j1 == n_units, fresh = entry && warp == KS_WARPS - 1;
      uint4 kx, vx, kt;
      {
        uint4 x[NT][KJ][2], turn[KJ][2];
        bool have[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const int col = nt * 8 + r, i = col / a.n_rep;
          const long long row = row0 + (long long)i * a.step;
          have[nt] = col < n_cols && row >= 0 && row < a.R;
          const __half* q = a.x + (size_t)(have[nt] ? row : 0) * a.ldx + (size_t)(g * a.n_rep + (have[nt] ? col - i * a.n_rep : 0)) * HD + c * 16;
#pragma unroll
          for (int j = 0; j < KJ; j++) { x[nt][j][0] = ld_128(q + j * 64); x[nt][j][1] = ld_128(q + j * 64 + 8); }
        }
        const bool turned = NEW && a.table;
        if (turned)
#pragma unroll
          for (int j = 0; j < KJ; j++) {
            const __half* from = a.table + (size_t)p0 * HD + c * 16 + j * 64;
            turn[j][0] = ld_128(from);
            turn[j][1] = ld_128(from + 8);
          }
        if (fresh) {
          const __half* k = a.x + (size_t)b * a.ldx + (size_t)(a.H + g) * HD + lane % (HD / 8) * 8;
          kx = ld_128(k);
          vx = ld_128(k + (size_t)a.c.G * HD);
          if (a.table) kt = ld_128(a.table + (size_t)p0 * HD + lane % (HD / 8) * 8);
        }
        if (n_tiles > 0) load(0, tile);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int j = 0; j < KJ; j++) {
            uint4 lo = x[nt][j][0], hi = x[nt][j][1];
            if (turned) { lo = kvq_rotate(lo, turn[j][0]); hi = kvq_rotate(hi, turn[j][1]); }
            if (!have[nt]) lo = hi = make_uint4(0, 0, 0, 0);
            ks_put(q_at + (nt * KJ + j) * 1024, lo);
            ks_put(q_at + (nt * KJ + j) * 1024 + 512, hi);
          }
      }
      asm volatile("" : "+r"(q_at)::"memory");  // what is read at q_at comes after
      // ---- the new token
      if (fresh) {
        constexpr int LPR = HD / 8;
        const int sub = lane % LPR;
        if (a.table) kx = kvq_rotate(kx, kt);
        uint2 kc, vc;
        __half2 scale;
        kvq_quantise<FMT, LPR>(kx, vx, kc, vc, scale);
        if (lane < LPR) {
          const size_t to = kvq_row(a.c, bt, p0, g);
          *reinterpret_cast<uint2*>(a.c.k + to * HD + sub * 8) = kc;
          *reinterpret_cast<uint2*>(a.c.v + to * HD + sub * 8) = vc;
          if (sub == 0) a.c.scales[to] = scale;
          __half2 h[4], w[4];
          kvq_widen<FMT>(kc.x, h[0], h[1]);
          kvq_widen<FMT>(kc.y, h[2], h[3]);
          kvq_widen<FMT>(vc.x, w[0], w[1]);
          kvq_widen<FMT>(vc.y, w[2], w[3]);
#pragma unroll
          for (int j = 0; j < 4; j++) { h[j] = __hmul2_rn(h[j], __low2half2(scale)); w[j] = __hmul2_rn(w[j], __high2half2(scale)); }
          *reinterpret_cast<uint4*>(&s_new[0][sub * 8]) = *reinterpret_cast<const uint4*>(h);
          *reinterpret_cast<uint4*>(&s_new[1][sub * 8]) = *reinterpret_cast<const uint4*>(w);
        }
        __syncwarp();
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < KJ * 2; j++) {
          const uint4 k = ld_128(&s_new[0][(j >> 1) * 64 + c * 16 + (j & 1) * 8]), q = ks_get(q_at + j * 512, 0);
          const uint32_t kw[4] = {k.x, k.y, k.z, k.w}, qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float2 k0 = h2_to_f2(kw[e]), q0 = h2_to_f2(qw[e]);
            s = fmaf(k0.x, q0.x, fmaf(k0.y, q0.y, s));
          }
        }
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        if (c == 0) { s_m[KS_WARPS][r] = s * a.scale2; s_l[KS_WARPS][r] = 1.f; }
      }

      // ---- the loop over tiles
      float o[NT][MT][4], m[NT][2], l[NT][2];
      int lim[NT][2];  // last position that the lane's columns of a score tile see
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int k = 0; k < MT; k++) o[nt][k][0] = o[nt][k][1] = o[nt][k][2] = o[nt][k][3] = 0.f;
#pragma unroll
        for (int e = 0; e < 2; e++) {
          m[nt][e] = -INFINITY;
          l[nt][e] = 0.f;
          lim[nt][e] = NEW ? T - 1 : (int)min((long long)T - 1, (long long)p0 + (nt * 8 + 2 * c + e) / a.n_rep);
        }
      }
      for (int i = 0; i < n_tiles; i++) {
        const Tile t = tile;
        if (i + 1 < n_tiles) load(i + 1, tile);
        const int t0 = t_lo + i * KS_UNIT + warp * 16;
        // scores
        float s[NT][4], s_[NT][4];  // in two chains of products
#pragma unroll
        for (int nt = 0; nt < NT; nt++) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = s_[nt][0] = s_[nt][1] = s_[nt][2] = s_[nt][3] = 0.f;
#pragma unroll
        for (int j = 0; j < KJ; j++) {
          const uint32_t w0[4] = {t.k[0][j].x, t.k[0][j].y, t.k[0][j].z, t.k[0][j].w}, w1[4] = {t.k[1][j].x, t.k[1][j].y, t.k[1][j].z, t.k[1][j].w};
          uint32_t qw[NT][8];
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            const uint4 lo = ks_get(q_at + (nt * KJ + j) * 1024, i), hi = ks_get(q_at + (nt * KJ + j) * 1024 + 512, i);
            qw[nt][0] = lo.x; qw[nt][1] = lo.y; qw[nt][2] = lo.z; qw[nt][3] = lo.w;
            qw[nt][4] = hi.x; qw[nt][5] = hi.y; qw[nt][6] = hi.z; qw[nt][7] = hi.w;
          }
#pragma unroll
          for (int e = 0; e < 4; e++) {
            __half2 a0, a1, a2, a3;
            kvq_widen<FMT>(w0[e], a0, a2);
            kvq_widen<FMT>(w1[e], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
              ks_mma(e & 1 ? s_[nt] : s[nt], ks_half2(a0), ks_half2(a1), ks_half2(a2), ks_half2(a3), qw[nt][2 * e], qw[nt][2 * e + 1]);
          }
        }
        const float ks0 = __low2float(t.s0) * a.scale2, ks1 = __low2float(t.s1) * a.scale2;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) { s[nt][0] += s_[nt][0]; s[nt][1] += s_[nt][1]; s[nt][2] += s_[nt][2]; s[nt][3] += s_[nt][3]; }
        bool over = false;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          s[nt][0] = t0 + r <= lim[nt][0] ? s[nt][0] * ks0 : -INFINITY;
          s[nt][1] = t0 + r <= lim[nt][1] ? s[nt][1] * ks0 : -INFINITY;
          s[nt][2] = t0 + r + 8 <= lim[nt][0] ? s[nt][2] * ks1 : -INFINITY;
          s[nt][3] = t0 + r + 8 <= lim[nt][1] ? s[nt][3] * ks1 : -INFINITY;
          over = over || fmaxf(s[nt][0], s[nt][2]) > m[nt][0] + 6.f || fmaxf(s[nt][1], s[nt][3]) > m[nt][1] + 6.f;
        }
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float top = fmaxf(s[nt][e], s[nt][e + 2]);
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
              top = fmaxf(top, m[nt][e]);
              const float fade = top == m[nt][e] ? 1.f : ex2(m[nt][e] - top);
              m[nt][e] = top;
              l[nt][e] *= fade;
#pragma unroll
              for (int k = 0; k < MT; k++) { o[nt][k][e] *= fade; o[nt][k][e + 2] *= fade; }
            }
        }
        uint32_t w[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          const float b0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], b1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
          const float e0 = ex2(s[nt][0] - b0), e1 = ex2(s[nt][1] - b1), e2 = ex2(s[nt][2] - b0), e3 = ex2(s[nt][3] - b1);
          l[nt][0] += e0 + e2;
          l[nt][1] += e1 + e3;
          w[nt][0] = ks_transpose(ks_half2(__floats2half2_rn(e0, e1)));
          w[nt][1] = ks_transpose(ks_half2(__floats2half2_rn(e2, e3)));
        }
        // outputs
        uint32_t p0_ = __byte_perm(t.sv0.x, t.sv0.y, 0x7632), p1_ = __byte_perm(t.sv1.x, t.sv1.y, 0x7632);
        if (NEW && t0 + 16 > T) {
          // The row behind the last is being written by another warp: new codes times the scale that was there could be an infinity, and that
          // times a weight of 0 a NaN.
          const int left = T - t0 - 2 * c;
          p0_ &= (left > 0 ? 0xFFFFu : 0u) | (left > 1 ? 0xFFFF0000u : 0u);
          p1_ &= (left > 8 ? 0xFFFFu : 0u) | (left > 9 ? 0xFFFF0000u : 0u);
        }
        const __half2 scale0 = *reinterpret_cast<const __half2*>(&p0_), scale1 = *reinterpret_cast<const __half2*>(&p1_);
#pragma unroll
        for (int e = 0; e < VB / 4; e++)
#pragma unroll
          for (int half = 0; half < 2; half++) {
            const uint32_t lo = __byte_perm(t.v[0][e], t.v[1][e], half ? 0x7362 : 0x5140), hi = __byte_perm(t.v[2][e], t.v[3][e], half ? 0x7362 : 0x5140);
            __half2 a0, a1, a2, a3;
            kvq_widen<FMT>(lo, a0, a1);
            kvq_widen<FMT>(hi, a2, a3);
            a0 = __hmul2_rn(a0, scale0); a1 = __hmul2_rn(a1, scale0);
            a2 = __hmul2_rn(a2, scale1); a3 = __hmul2_rn(a3, scale1);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
              ks_mma(o[nt][2 * e + half], ks_half2(a0), ks_half2(a1), ks_half2(a2), ks_half2(a3), w[nt][0], w[nt][1]);
          }
      }

      // ---- the warps' sums meet 
      float* so = reinterpret_cast<float*>(ks_raw);  // [warp][column][hd]
      __syncthreads();
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float sum = l[nt][e];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          const int col = nt * 8 + 2 * c + e;
          if (r == 0) { s_m[warp][col] = m[nt][e]; s_l[warp][col] = sum; }
          float* to = so + ((size_t)warp * COLS + col) * HD + r * VB;
#pragma unroll
          for (int k = 0; k < MT; k++) *reinterpret_cast<float2*>(to + 2 * k) = make_float2(o[nt][k][e], o[nt][k][e + 2]);
        }
      __syncthreads();
      const bool whole = j0 == 0 && j1 == n_units;
      float* part = whole ? nullptr : a.part + (size_t)kvq_slot(blockIdx.x, j0 == 0) * Cfg::PART;
      auto store = [&](int idx, const float (&x)[4]) {  // four finished values of a column
        const int col = idx / HD, i = col / a.n_rep;
        const long long row = row0 + (long long)i * a.step;
        if (col >= n_cols || row < 0 || row >= a.R) return;
        // zeros where there is nothing to see; where all scores are -inf (an infinite query) the sum is 0 and the row NaN, as a softmax is
        const bool outside = !NEW && (bt == nullptr || (long long)p0 + i >= a.limit || (long long)p0 + i < 0);
        const __half2 h0 = __floats2half2_rn(outside ? 0.f : x[0], outside ? 0.f : x[1]), h1 = __floats2half2_rn(outside ? 0.f : x[2], outside ? 0.f : x[3]);
        *reinterpret_cast<uint2*>(a.out + (size_t)row * a.ldo + (size_t)(g * a.n_rep + col % a.n_rep) * HD + idx % HD) = make_uint2(ks_half2(h0), ks_half2(h1));
      };
      for (int idx = tid * 4; idx < COLS * HD; idx += KS_THREADS * 4) {
        const int col = idx / HD;
        float top = NEW && entry ? s_m[KS_WARPS][col] : -INFINITY;
#pragma unroll
        for (int w = 0; w < KS_WARPS; w++) top = fmaxf(top, s_m[w][col]);
        const float base = top == -INFINITY ? 0.f : top;
        float x[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll
        for (int w = 0; w < KS_WARPS; w++) {
          const float f = ex2(s_m[w][col] - base);
          const float4 y = *reinterpret_cast<const float4*>(so + (size_t)w * COLS * HD + idx);
          sum = fmaf(s_l[w][col], f, sum);
          x[0] = fmaf(y.x, f, x[0]); x[1] = fmaf(y.y, f, x[1]); x[2] = fmaf(y.z, f, x[2]); x[3] = fmaf(y.w, f, x[3]);
        }
        if (NEW && entry) {
          const float f = ex2(s_m[KS_WARPS][col] - base);
          const uint2 y = *reinterpret_cast<const uint2*>(&s_new[1][idx % HD]);
          const float2 y0 = h2_to_f2(y.x), y1 = h2_to_f2(y.y);
          sum += f;
          x[0] = fmaf(y0.x, f, x[0]); x[1] = fmaf(y0.y, f, x[1]); x[2] = fmaf(y1.x, f, x[2]); x[3] = fmaf(y1.y, f, x[3]);
        }
        if (whole) {
          const float inv = __fdiv_rn(1.f, sum);
          x[0] *= inv; x[1] *= inv; x[2] *= inv; x[3] *= inv;
          store(idx, x);
        } else {
          __stcg(reinterpret_cast<float4*>(part + idx), make_float4(x[0], x[1], x[2], x[3]));
          if (idx % HD == 0) { __stcg(part + COLS * HD + col, top); __stcg(part + COLS * HD + COLS + col, sum); }
        }
      }
      if (whole) { __syncthreads(); continue; }
      // ---- pieces of a (sequence, kv head) that several CTAs, from c_lo on, share: the last to arrive adds them up in this order.  Many are added up in
      // groups of neighbours first, as these are done: one CTA reads 30 pieces in 10 us.
      const long long begin = item + Cfg::FIXED, last = begin + n_units - 1;
      const int c_lo = kvq_owner(total, ctas, begin), pieces = kvq_owner(total, ctas, last) - c_lo + 1;
      auto arrive = [&](unsigned int* ticket, int of) -> bool {  // whether this CTA is the last
        __syncthreads();
        if (tid == 0) {
          __threadfence();
          s_ticket = atomicAdd(ticket, 1u);
          if (s_ticket == (unsigned)(of - 1)) *ticket = 0;
          __threadfence();
        }
        __syncthreads();
        return s_ticket == (unsigned)(of - 1);
      };
      auto piece = [&](int p) -> float* { return a.part + (size_t)kvq_slot(c_lo + p, p == 0) * Cfg::PART; };
      // groups of four values of a thread; pieces whose loads are in flight together
      constexpr int NI = COLS * HD / (KS_THREADS * 4), BATCH = NI > 2 ? 2 : NI > 1 ? 4 : 8;
      float x[NI][4], top[NI], sum[NI];
      auto add_up = [&](int from, int to, int step) {
#pragma unroll
        for (int e = 0; e < NI; e++) { x[e][0] = x[e][1] = x[e][2] = x[e][3] = sum[e] = 0.f; top[e] = -INFINITY; }
#pragma unroll 1
        for (int p = from; p < to; p += BATCH * step) {
          float4 y[BATCH][NI];
          float pm[BATCH][NI], pl[BATCH][NI];
#pragma unroll
          for (int k = 0; k < BATCH; k++) {
            const float* src = piece(p + k * step < to ? p + k * step : from);
#pragma unroll
            for (int e = 0; e < NI; e++) {
              const int idx = (tid + e * KS_THREADS) * 4;
              y[k][e] = __ldcg(reinterpret_cast<const float4*>(src + idx));
              pm[k][e] = __ldcg(src + COLS * HD + idx / HD);
              pl[k][e] = __ldcg(src + COLS * HD + COLS + idx / HD);
            }
          }
#pragma unroll
          for (int k = 0; k < BATCH; k++)
#pragma unroll
            for (int e = 0; e < NI; e++) {
              if (p + k * step >= to) continue;
              const float then = fmaxf(top[e], pm[k][e]), base = then == -INFINITY ? 0.f : then, fade = ex2(top[e] - base), f = ex2(pm[k][e] - base);
              top[e] = then;
              sum[e] = sum[e] * fade + pl[k][e] * f;
              x[e][0] = x[e][0] * fade + y[k][e].x * f;
              x[e][1] = x[e][1] * fade + y[k][e].y * f;
              x[e][2] = x[e][2] * fade + y[k][e].z * f;
              x[e][3] = x[e][3] * fade + y[k][e].w * f;
            }
        }
      };
      const KsGroup group = ks_group((int)blockIdx.x - c_lo, pieces, c_lo);
      if (group.ticket >= 0) {
        if (!arrive(&a.tickets[group.ticket], group.to - group.from)) continue;
        add_up(group.from, group.to, 1);
        __syncthreads();  // all have read what is written over now
        float* dst = piece(group.from);
#pragma unroll
        for (int e = 0; e < NI; e++) {
          const int idx = (tid + e * KS_THREADS) * 4;
          __stcg(reinterpret_cast<float4*>(dst + idx), make_float4(x[e][0], x[e][1], x[e][2], x[e][3]));
          if (idx % HD == 0) { __stcg(dst + COLS * HD + idx / HD, top[e]); __stcg(dst + COLS * HD + COLS + idx / HD, sum[e]); }
        }
      }
      if (!arrive(&a.tickets[ks_last_ticket(gridDim.x, c_lo)], ks_groups(pieces, group.step))) continue;
      add_up(0, pieces, group.step);
#pragma unroll
      for (int e = 0; e < NI; e++) {
        const float inv = __fdiv_rn(1.f, sum[e]);
        x[e][0] *= inv; x[e][1] *= inv; x[e][2] *= inv; x[e][3] *= inv;
        store((tid + e * KS_THREADS) * 4, x[e]);
      }
      __syncthreads();
    }
    at += (long long)span * a.c.G;
  }
}

static inline int ks_ctas(const jg_dev* dev) { return KS_CTAS * dev->sm_count; }  // that a device runs at once; twice as many tickets: jg_kvq_ticket_bytes
static inline int ks_slots(const jg_dev* dev) { return 2 * ks_ctas(dev); }  // pieces in the workspace
static inline size_t ks_part_floats(int hd) { return hd == 64 ? KsCfg<64, 4>::PART : KsCfg<128, 3>::PART; }

template <int FMT, int HD, int NT, bool NEW>
static int launch_split(jg_dev* dev, const KvqSplitArgs& a) {
  auto kern = kvq_split_kernel<FMT, HD, NT, NEW>;
  using Cfg = KsCfg<HD, NT>;
  const size_t smem = Cfg::MERGE;
  static bool attr_set[8] = {};
  if (!attr_set[dev->ordinal & 7]) {
    JG_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    attr_set[dev->ordinal & 7] = true;
  }
  const int ctas = NT == 1 ? ks_ctas(dev) : 2 * dev->sm_count;  // that run at once
  const long long most = (long long)a.B * a.c.G * ((a.c.max_ctx + KS_UNIT - 1) / KS_UNIT);
  return jg_launch(dev, NEW ? "kvq_decode" : "kvq_attn", kern, dim3((unsigned)(most < ctas ? most : ctas)), dim3(KS_THREADS), smem, a);
}
#endif
