// Arguments of the norm-and-rotation kernels (esa_rotary.hip).
#pragma once
#include "esa_internal.hpp"

namespace esa {

struct RotaryArgs {
  const void *q, *k, *v;  // rows in (v: append only)
  void *qo, *ko, *vo;     // rows out: q, k; append: q and the two caches; backward: dq, dk
  const void *gq, *gk;    // backward: gradients of the rotated rows
  int64_t qsb, qsh, qss, ksb, ksh, kss, vsb, vsh, vss;
  int64_t qosb, qosh, qoss, kosb, kosh, koss, vosb, vosh, voss;
  int64_t gqsb, gqsh, gqss, gksb, gksh, gkss;
  const void *wq, *wk;  // gains, or NULL (1)
  void *dwq, *dwk;
  const double* inv_freq;
  const int64_t* pos;
  int64_t pos_sb;
  int H, Hkv, n, D, rd, kv_len;
  int elem, welem, vec;  // vec: elements a lane holds
  int interleaved;
  float eps;
  // the grid: tiles of 256 / (lanes a row) of all sequences' tokens, heads (q, k
  // and, to append, v) in splits; grid_tiles workgroups walk the n_tiles tiles
  int lanes, tokens, n_tiles, grid_tiles;
  int side;  // heads of a token side by side in a workgroup: 1 or 2
  int heads, heads_per_split, n_splits;
  FastDiv div_n, div_half;
  float* partial;  // backward: [grid_tiles n_splits][2][D] sums of the gains' gradients
};

hipError_t launch_rotary(const RotaryArgs& a, int mode, hipStream_t stream);

}  // namespace esa
