// Internal interface between csrc/paged_attention.cu (the entry points, the per-sequence kernel) and
// csrc/paged_prefix.cu (the tcgen05 kernel of a prefix that the batch shares).
#pragma once

#include <cuda.h>

#include "paged.cuh"

namespace b2d {

constexpr int kMaxParts = 32;      // partials of the prefix launch

struct PagedAttnArgs {
  const void* q; int64_t sq_b, sq_t, sq_h;
  const int32_t* table; int64_t ld_table;
  const int32_t* seqlens;
  const int32_t* prefix_table;
  void* out; int64_t so_b, so_t, so_h;
  b2d_paged_kv kv;
  PageDiv div;
  int pages_per_seq, prefix_len, B, T, H, G, rows;   // rows = T G
  float scale_log2;
  int shared;       // positions [0, shared) are the prefix launch's (0: there is none)
  int cs, ncl;      // CTAs of a cluster; clusters of one (sequence, KV head, row tile)
  int tiles;        // row tiles
  int nparts;       // partials of the prefix launch
  int parts;        // nparts + (ncl > 1 ? ncl : 0): partials in the workspace
  int out_f32, after_prefix;
  int box_rows;     // key rows of a tensor copy; 0: the pages take cp.async
  float* acc;       // [parts][B T H][D] unnormalised, row = (b T + t) H + h
  float* ml;        // [parts][B T H][2] m (log2 domain), l
};

// Tensor maps of the pools: [pages][heads][slots][D], boxes of 64 elements x box_rows slots.
struct PoolMaps {
  CUtensorMap k, v;
};

// The prefix [0, a.shared) for the rows of all sequences on the 5th-generation tensor cores: a.nparts splits
// over the keys, each leaving (O, m, l) per row in a.acc / a.ml. Needs a.box_rows > 0 and a.shared % 64 == 0.
int launch_prefix_tc5(const PoolMaps& maps, const PagedAttnArgs& a, bool pdl, cudaStream_t stream);

}  // namespace b2d
