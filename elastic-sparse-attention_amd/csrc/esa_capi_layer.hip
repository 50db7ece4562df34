// C ABI of the operators around an attention layer's calls (include/esa.h):
// argument checks on the host, then kernel launches.
#include <algorithm>
#include <cmath>

#include "esa.h"
#include "esa_rotary.hpp"

using namespace esa;

namespace {

bool aligned(const void* ptr, size_t a) { return ((uintptr_t)ptr % a) == 0; }

bool dtype_ok(esa_dtype t) { return t == ESA_F32 || t == ESA_BF16 || t == ESA_F16; }

constexpr int kRotFwd = 0, kRotAppend = 1, kRotBwd = 2;
// workgroups of the norm-and-rotation backward, at most: four a CU; each
// writes one row of partial sums
constexpr int kRotBwdGrid = 1024;

esa_status rotary_check(const esa_rotary_args* a) {
  if (!a) return ESA_ERR_NULL;
  if (!dtype_ok(a->dtype) || !dtype_ok(a->weight_dtype)) return ESA_ERR_DTYPE;
  if (a->batch < 0 || a->num_heads < 1 || a->num_kv_heads < 1 || a->seq_len < 0 ||
      a->head_dim < 1 || a->rotary_dim < 1 || a->rotary_dim > a->head_dim ||
      a->interleaved < 0 || a->interleaved > 1 || a->position_stride_b < 0)
    return ESA_ERR_SHAPE;
  if (a->head_dim % 4 != 0 || a->head_dim > 256 || a->rotary_dim % 8 != 0)
    return ESA_ERR_UNSUPPORTED;
  if (!(a->eps >= 0.f) || !std::isfinite(a->eps)) return ESA_ERR_SHAPE;
  // rows and tiles are counted in int32
  if (a->num_heads > (1 << 20) || a->num_kv_heads > (1 << 20) ||
      (int64_t)a->batch * a->seq_len >= (int64_t(1) << 31))
    return ESA_ERR_SHAPE;
  return ESA_OK;
}

// elements a lane holds: 16 bytes, or 8 where they do not fit the rotation
int rotary_vec(const esa_rotary_args* a) {
  if (a->dtype == ESA_F32) return 4;
  return a->head_dim % 8 == 0 && (a->interleaved || a->rotary_dim % 16 == 0) ? 8 : 4;
}

// Tokens of a tile and the split of the heads: eight tokens and all heads a
// workgroup, halved and then split until the grid holds `want` workgroups (a
// call of few tokens runs its heads side by side: one token of 40 heads at
// head_dim 128 in three workgroups).
void rotary_grid(RotaryArgs& g, int batch, bool append, bool bwd) {
  const int want = 1024;
  g.heads = g.H + g.Hkv + (append ? g.Hkv : 0);
  g.log_t = 3;
  auto tiles = [&] { return (int64_t)batch * ((g.n + (1 << g.log_t) - 1) >> g.log_t); };
  while (g.log_t > 0 && tiles() < want) --g.log_t;
  const int lanes = (g.D + g.vec - 1) / g.vec;
  int lpr = 8;
  while (lpr < lanes) lpr *= 2;
  const int pass = std::max(1, 256 / lpr >> g.log_t);  // heads a pass takes
  g.tiles_per_seq = (g.n + (1 << g.log_t) - 1) >> g.log_t;
  g.n_tiles = (int)tiles();
  const int most = (g.heads + pass - 1) / pass;
  const int split = (int)std::min<int64_t>(most, std::max<int64_t>(1, want / g.n_tiles));
  g.heads_per_split = ((g.heads + split - 1) / split + pass - 1) / pass * pass;
  g.heads_per_split = std::min(g.heads_per_split, g.heads);
  g.n_splits = (g.heads + g.heads_per_split - 1) / g.heads_per_split;
  // (a grid dimension holds fewer than 2^32 work-items: 256 a workgroup)
  g.grid_tiles = std::min(g.n_tiles, bwd ? kRotBwdGrid : 1 << 23);
  g.div_tiles = make_fast_div((uint32_t)g.tiles_per_seq);
  g.div_half = make_fast_div((uint32_t)(g.rd / 2));
  g.div_heads = make_fast_div((uint32_t)g.heads_per_split);
}

RotaryArgs rotary_args(const esa_rotary_args* a, int mode) {
  RotaryArgs g{};
  g.q = a->q; g.k = a->k; g.v = a->v;
  g.qo = a->q_out; g.ko = a->k_out; g.vo = a->v_out;
  g.gq = a->q_grad; g.gk = a->k_grad;
  g.qsb = a->q_stride_b; g.qsh = a->q_stride_h; g.qss = a->q_stride_s;
  g.ksb = a->k_stride_b; g.ksh = a->k_stride_h; g.kss = a->k_stride_s;
  g.vsb = a->v_stride_b; g.vsh = a->v_stride_h; g.vss = a->v_stride_s;
  g.qosb = a->q_out_stride_b; g.qosh = a->q_out_stride_h; g.qoss = a->q_out_stride_s;
  g.kosb = a->k_out_stride_b; g.kosh = a->k_out_stride_h; g.koss = a->k_out_stride_s;
  g.vosb = a->v_out_stride_b; g.vosh = a->v_out_stride_h; g.voss = a->v_out_stride_s;
  g.gqsb = a->q_grad_stride_b; g.gqsh = a->q_grad_stride_h; g.gqss = a->q_grad_stride_s;
  g.gksb = a->k_grad_stride_b; g.gksh = a->k_grad_stride_h; g.gkss = a->k_grad_stride_s;
  g.wq = a->q_weight; g.wk = a->k_weight;
  g.dwq = a->q_weight_grad; g.dwk = a->k_weight_grad;
  g.inv_freq = a->inv_freq;
  g.pos = a->positions; g.pos_sb = a->position_stride_b;
  g.H = a->num_heads; g.Hkv = a->num_kv_heads; g.n = a->seq_len; g.D = a->head_dim;
  g.rd = a->rotary_dim; g.kv_len = a->kv_len;
  g.elem = a->dtype; g.welem = a->weight_dtype; g.vec = rotary_vec(a);
  g.interleaved = a->interleaved;
  g.eps = a->eps;
  // a token's heads lie side by side ([B, L, H, D] memory)
  g.heads_fast = a->q_stride_h < a->q_stride_s;
  rotary_grid(g, a->batch, mode == kRotAppend, mode == kRotBwd);
  return g;
}

struct RotaryTensor {
  const void* p;
  int64_t sb, sh, ss;
};

esa_status rotary_run(const esa_rotary_args* a, int mode, void* workspace, size_t ws_bytes,
                      void* stream) {
  const esa_status s = rotary_check(a);
  if (s != ESA_OK) return s;
  if (mode == kRotAppend && a->kv_len < 1) return ESA_ERR_SHAPE;
  if (a->batch == 0 || a->seq_len == 0) return ESA_OK;
  RotaryTensor ts[7] = {{a->q, a->q_stride_b, a->q_stride_h, a->q_stride_s},
                        {a->k, a->k_stride_b, a->k_stride_h, a->k_stride_s},
                        {a->q_out, a->q_out_stride_b, a->q_out_stride_h, a->q_out_stride_s},
                        {a->k_out, a->k_out_stride_b, a->k_out_stride_h, a->k_out_stride_s}};
  int n = 4;
  if (mode == kRotAppend) {
    ts[n++] = {a->v, a->v_stride_b, a->v_stride_h, a->v_stride_s};
    ts[n++] = {a->v_out, a->v_out_stride_b, a->v_out_stride_h, a->v_out_stride_s};
  } else if (mode == kRotBwd) {
    ts[n++] = {a->q_grad, a->q_grad_stride_b, a->q_grad_stride_h, a->q_grad_stride_s};
    ts[n++] = {a->k_grad, a->k_grad_stride_b, a->k_grad_stride_h, a->k_grad_stride_s};
  }
  if (!a->inv_freq || !a->positions) return ESA_ERR_NULL;
  const int vec = rotary_vec(a);
  const size_t bytes = vec * (a->dtype == ESA_F32 ? 4 : 2);
  for (int i = 0; i < n; ++i) {
    if (!ts[i].p) return ESA_ERR_NULL;
    if (!aligned(ts[i].p, bytes) || ts[i].sb % vec || ts[i].sh % vec || ts[i].ss % vec)
      return ESA_ERR_ALIGN;
  }
  RotaryArgs g = rotary_args(a, mode);
  if (mode == kRotBwd && (a->q_weight_grad || a->k_weight_grad)) {
    const size_t need = (size_t)g.grid_tiles * g.n_splits * 2 * g.D * sizeof(float);
    if (!workspace) return ESA_ERR_NULL;
    if (!aligned(workspace, 16)) return ESA_ERR_ALIGN;
    if (ws_bytes < need) return ESA_ERR_CAPACITY;
    g.partial = (float*)workspace;
  }
  return launch_rotary(g, mode, (hipStream_t)stream) == hipSuccess ? ESA_OK : ESA_ERR_HIP;
}

}  // namespace

extern "C" {

esa_status esa_qk_norm_rope_fwd(const esa_rotary_args* a, void* stream) {
  return rotary_run(a, kRotFwd, nullptr, 0, stream);
}

esa_status esa_qk_norm_rope_append(const esa_rotary_args* a, void* stream) {
  return rotary_run(a, kRotAppend, nullptr, 0, stream);
}

esa_status esa_qk_norm_rope_bwd_workspace_size(const esa_rotary_args* a, size_t* bytes) {
  if (!bytes) return ESA_ERR_NULL;
  const esa_status s = rotary_check(a);
  if (s != ESA_OK) return s;
  *bytes = 0;
  if (a->batch == 0 || a->seq_len == 0 || (!a->q_weight_grad && !a->k_weight_grad)) return ESA_OK;
  const RotaryArgs g = rotary_args(a, kRotBwd);
  *bytes = (size_t)g.grid_tiles * g.n_splits * 2 * g.D * sizeof(float);
  return ESA_OK;
}

esa_status esa_qk_norm_rope_bwd(const esa_rotary_args* a, void* workspace, size_t workspace_bytes,
                                void* stream) {
  return rotary_run(a, kRotBwd, workspace, workspace_bytes, stream);
}

}  // extern "C"
