// The tensor-core form of attention over the 8-bit cache: its arguments and the size of its workspace (kvquant_chunk.cu).
#pragma once
#include "kvquant.cuh"
#include "kvquant_line.h"

struct KvqChunkArgs {
  KvqLayer c;
  const __half* q;
  __half* out;
  const int32_t* pos;
  const int32_t* count;
  const int32_t* first;
  const int32_t* seq;
  int ldq, ldo, R, B, n_rep, max_count, step;
  int max_tiles;          // items that max_count positions make
  float scale2;           // log2 e / sqrt(hd)
  float* part;            // [kc_slots][kc_part_floats]
  unsigned int* tickets;  // [CTAs], zero between launches
  int* err;
};

static inline int kc_ctas(const jg_dev* dev) { return dev->sm_count < 512 ? dev->sm_count : 512; }
static inline int kc_slots(const jg_dev* dev) { return 2 * kc_ctas(dev); }  // pieces in the workspace
__host__ __device__ constexpr size_t kc_part_floats(int hd) { return (size_t)KC_ROWS * (hd + 2); }  // outputs, maxima, sums

int kvq_chunk(jg_dev* dev, int format, int hd, const KvqChunkArgs& a);
