// Internal interface between csrc/paged_attention.cu (the entry points, the streaming kernel, the combine) and
// csrc/paged_prefix.cu (the tcgen05 kernel of a prefix that the batch shares).
#pragma once

#include <cuda.h>

#include "paged.cuh"

namespace b2d {

constexpr int kMaxParts = 32;      // partials of the tcgen05 prefix launch

struct PagedAttnArgs {
  const void* q; int64_t sq_b, sq_t, sq_h;
  const int32_t* table; int64_t ld_table;
  const int32_t* seqlens;
  const int32_t* prefix_table;
  void* out; int64_t so_b, so_t, so_h;
  b2d_paged_kv kv;
  PageDiv div;
  int pages_per_seq, prefix_len, B, T, H, G, rows;   // rows = T G: query vectors of a sequence and KV head
  int inv_g;        // 2^16 / G, rounded up
  float scale_log2;
  int shared;       // positions [0, shared) are computed once for the batch (0: none are)
  int nparts;       // partials of the tcgen05 prefix launch (0: the streaming kernel takes the prefix)
  int splits;       // its CTAs per (row tiles, KV head)
  int ctas;         // CTAs of the streaming launch
  int whole;        // a CTA takes whole (sequence, KV head, row tile) units
  int out_f32, out_vec, after_prefix;
  int box_rows;     // key rows of a tensor copy; 0: the pages take cp.async
  // Workspace entries of D unnormalised fp32 sums and (m in the log2 domain, l); R = B T H rows (b T + t) H + h:
  // [nparts][R] of the tcgen05 launch, then, where a prefix joins them, [R] whole own and [R] whole prefix
  // parts; from slot0 on [ctas][2][row tile] of units that several CTAs share
  int64_t slot0;
  float* acc;
  float* ml;
};

// Tensor maps of the pools: [pages][heads][slots][D], boxes of 64 elements x box_rows slots.
struct PoolMaps {
  CUtensorMap k, v;
};

// The prefix [0, a.shared) for the rows of all sequences on the 5th-generation tensor cores: a.splits CTAs over
// the keys per (256 rows, KV head), leaving a.nparts entries per row. Needs a.box_rows > 0, a.shared % 64 == 0.
int launch_prefix_tc5(const PoolMaps& maps, const PagedAttnArgs& a, bool pdl, cudaStream_t stream);

}  // namespace b2d
