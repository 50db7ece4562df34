// C ABI of the operators around an attention layer's calls (include/esa.h):
// argument checks on the host, then kernel launches.
#include <algorithm>
#include <cmath>

#include "esa.h"
#include "esa_rotary.hpp"
#include "esa_sink.hpp"

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

// A workgroup takes a tile of tokens (256 lanes' worth of rows) through all
// heads; the heads are split over workgroups while the tiles alone make fewer
// than 512 (two a CU), down to one head each (one token of 40 heads: 40
// workgroups).  Two prompts of 500, 48 heads of 128: 13.2 us at 512 workgroups,
// 15.1 at 256, 19.1 at 128; and where the tiles are about 512 already a second
// split only forms their angles again (8192 tokens, 40 heads, backward: 56 us
// at 512, 65 at 1024).
void rotary_grid(RotaryArgs& g, int batch, bool append, bool bwd) {
  g.heads = g.H + g.Hkv + (append ? g.Hkv : 0);
  g.lanes = 8;
  while (g.lanes * g.vec < g.D) g.lanes *= 2;
  const int tok = 256 / g.lanes;
  // Where a token's heads are side by side in memory and the rows do not fit the
  // 256 MiB last-level cache, two lane groups take two heads of a token instead
  // of one of two tokens: twice the bytes at an address (40 heads of 128, bf16,
  // views of one projection, one and two: 32768 tokens 171 and 160 us, 16384 82
  // and 78, but 4096 26 and 27; the backward's five streams gain nothing, 256
  // and 271).
  const int es = g.elem == ESA_F32 ? 4 : 2;
  g.side = !bwd && g.qsh < g.qss && g.ksh < g.kss &&
                   2 * es * (double)batch * g.n * g.heads * g.D > double(256 << 20) ? 2 : 1;
  g.tokens = batch * g.n;
  g.n_tiles = (int)(((int64_t)g.tokens + tok - 1) / tok);
  const int64_t split = std::min<int64_t>(g.heads, (511 + g.n_tiles) / g.n_tiles);
  g.heads_per_split = ((int)((g.heads + split - 1) / split) + g.side - 1) / g.side * g.side;
  g.n_splits = (g.heads + g.heads_per_split - 1) / g.heads_per_split;
  // (a grid dimension holds fewer than 2^32 work-items: 256 a workgroup)
  g.grid_tiles = std::min(g.n_tiles, bwd ? kRotBwdGrid : 1 << 23);
  g.div_n = make_fast_div((uint32_t)g.n);
  g.div_half = make_fast_div((uint32_t)(g.rd / 2));
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

constexpr int64_t kMaxKeys = int64_t(1) << 26;      // positions and rows are int32
constexpr int64_t kMaxGrid = int64_t(1) << 24;      // workgroups of 256 work-items

// 16-byte rows: base and strides
esa_status sink_rows_ok(const void* p, int64_t sb, int64_t sh, int64_t ss, int elems) {
  if (!aligned(p, 16) || sb % elems || sh % elems || ss % elems) return ESA_ERR_ALIGN;
  return ESA_OK;
}

// a stage's rows lie within 2 GiB of its first one
bool stage_span_ok(int64_t stride, int es) {
  return stride >= 0 && stride < (int64_t(1) << 31) / (128 * es);
}

// The checks that the forward and the backward share.
esa_status sink_check(esa_dtype dtype, int32_t batch, int32_t heads, int32_t kv_heads,
                      int32_t q_len, int32_t kv_len, int32_t head_dim, float sm_scale,
                      const esa_window* w) {
  if (!w) return ESA_ERR_NULL;
  if (!dtype_ok(dtype)) return ESA_ERR_DTYPE;
  if (batch < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || q_len < 0 ||
      kv_len < 1 || head_dim < 1 || w->window < 1 || w->sinks < 0 || w->position_stride_b < 0)
    return ESA_ERR_SHAPE;
  if (q_len > kMaxKeys || kv_len > kMaxKeys || (!w->positions && q_len > kv_len))
    return ESA_ERR_SHAPE;
  const int epc = dtype == ESA_F32 ? 4 : 8;
  if (head_dim > 128 || head_dim % epc != 0) return ESA_ERR_UNSUPPORTED;
  if (!(sm_scale > 0.f) || !std::isfinite(sm_scale)) return ESA_ERR_UNSUPPORTED;
  if ((int64_t)batch * heads * ((q_len + 127) / 128) >= kMaxGrid ||
      (int64_t)batch * kv_heads * ((kv_len + 127) / 128) >= kMaxGrid)
    return ESA_ERR_SHAPE;
  return ESA_OK;
}

void sink_pattern(SinkArgs& g, const esa_window* w) {
  g.window = std::min(w->window, g.kv_len);
  // (a window over the whole cache hides nothing that sinks could show)
  g.sinks = g.window >= g.kv_len ? 0 : std::min(w->sinks, g.kv_len);
  g.pos = w->positions;
  g.pos_sb = w->position_stride_b;
  g.first = w->first_key;
  g.nqb = (g.q_len + 127) / 128;
}

// Which forward kernel, and into how many key ranges side by side.
//
// Few rows against many keys take the decode kernel (row tiles of 16 over the
// heads that share a kv head, the keys cut into ranges), others the forward's
// 128-row blocks, which walk their keys one after the other; blocks that leave
// CUs idle, or of which a few walk far more keys than the rest (a whole
// sequence's last rows), are cut into ranges too.  All are estimated.
//   decode: (tile, key) pairs a microsecond, after 8 us
//   blocks: a CU with 1, 2, .. of them walks a key of all in `walk` us (16-bit
//     128 dims: 158 us for two of 4227 keys each, 2110 for 8192 blocks, three a
//     CU; float32 gains nothing from a second), after 6 us; ranges add 10 and
//     their float32 parts, written and read at 4 TB/s
// Measured, decode against blocks (not cut): bf16, head_dim 128, 32 heads on 8,
// window 4096, one sequence, 1 / 16 / 64 rows 13 / 17 / 37 us against 94 / 96 /
// 99; 8 sequences, 4 / 16 / 32 rows 33 / 96 / 153 against 107 / 107 / 108; 64
// sequences, window 1024, 8 / 16 / 32 rows 82 / 157 / 306 against 149 / 147 /
// 147; head_dim 64, 64 sequences, 8 / 16 rows 46 / 84 against 58 / 59; float32,
// 16 sequences, 16 heads on 4 of 64, window 2048, 16 / 32 / 64 rows 67 / 83 / 134
// against 160 / 161 / 170; 8 sequences, 8 heads on 2 of 128, window 1024, 64 rows
// 57 against 162.  Blocks whole and cut (ranges): 2048 rows over 32768 keys, 4
// heads on one of 128 866 and 165 us (12); 1024 rows, 32 heads on 8 875 and 579
// (3); 512 rows, window 4096 118 and 68 (4); a sequence of 4096, 8 heads on 2 120
// and 79 (4); 2048 rows, 32 heads, window 4096 176 and 202 (2).
//
// Key ranges of the decode kernel: as many as make 512 workgroups (two a CU:
// with 1024 a 64-sequence step took 191 us against 184, four long sequences 102
// against 94), each of at least 128 keys, 32 a wave (one sequence over 1028
// keys: 9.9 us with 128, 11.3 with 256).
void sink_fwd_plan(SinkArgs& g) {
  const bool f32 = g.elem == ESA_F32, narrow = g.d_real <= 64;
  const int64_t rows = (int64_t)g.B * g.H * g.q_len;
  const int64_t tiles = (int64_t)g.B * g.Hkv * (((int64_t)g.groups * g.q_len + 15) / 16);
  const int64_t blocks = (int64_t)g.B * g.H * g.nqb;
  // the keys that a tile's, a block's rows walk, at most; a block on average
  // (whole sequences start with few)
  const int64_t seen = (int64_t)g.window + g.sinks;
  const int64_t tile_keys = std::min<int64_t>(g.kv_len, seen + std::min(g.q_len, 16));
  const double keys = (double)std::min<int64_t>(g.kv_len, seen + std::min(g.q_len, 128));
  const double mean = g.pos ? keys
                            : std::min(keys, 128.0 + g.sinks +
                                                 g.window * (1.0 - 0.5 * g.window / g.kv_len));
  const double rate = f32 ? (narrow ? 13000.0 : 4900.0) : narrow ? 27000.0 : 13500.0;
  static const double walks[3][4] = {{0.0265, 0.0374, 0.048, 0}, {0.0209, 0.0286, 0.0376, 0.049},
                                     {0.08, 0, 0, 0}};
  const double* walk = walks[f32 ? 2 : narrow ? 1 : 0];
  const int64_t fit = f32 ? 1 : narrow ? 4 : 3;  // blocks of a CU at a time
  const double scale = f32 && !narrow ? 1.8 : 1.0;
  auto blocks_time = [&](int64_t c) {
    const int64_t x = (blocks * c + 255) / 256;
    const double all = (double)(x / fit) * walk[fit - 1] + (x % fit ? walk[x % fit - 1] : 0.0);
    const double parts = c > 1 ? 10.0 + (double)rows * c * (narrow ? 64 : 128) * 8 / 4.0e6 : 0.0;
    return 6.0 + scale / (double)c * std::max(keys * walk[std::min(x, fit) - 1], mean * all) + parts;
  };
  const bool few = rows < kMaxGrid / 4;  // (a row's index fits 32 bits, its join a grid)
  g.splits = 1;
  double best = blocks_time(1);
  for (int64_t c = 2; few && c <= 64 && keys / c >= 256 && blocks * c <= 2048; ++c) {
    const double t = blocks_time(c);
    if (t < best) {
      best = t;
      g.splits = (int)c;
    }
  }
  g.decode = few && (tiles * (double)tile_keys / rate + 8.0 < best ||
                     (int64_t)g.groups * g.q_len <= 16);
  if (g.decode)
    g.splits = (int)std::min<int64_t>((tile_keys + 127) / 128, std::max<int64_t>(1, 512 / tiles));
  if (few) g.row_tiles = (g.groups * g.q_len + 15) / 16;
}

SinkArgs sink_fwd_args(const esa_fwd_args* a, const esa_window* w) {
  SinkArgs g{};
  g.q = a->q; g.k = a->k; g.v = a->v; g.o = a->o; g.lse = a->lse;
  g.qsb = a->q_stride_b; g.qsh = a->q_stride_h; g.qss = a->q_stride_s;
  g.ksb = a->k_stride_b; g.ksh = a->k_stride_h; g.kss = a->k_stride_s;
  g.vsb = a->v_stride_b; g.vsh = a->v_stride_h; g.vss = a->v_stride_s;
  g.osb = a->o_stride_b; g.osh = a->o_stride_h; g.oss = a->o_stride_s;
  g.lsb = a->lse_stride_b; g.lsh = a->lse_stride_h;
  g.B = a->batch; g.H = a->num_heads; g.Hkv = a->num_kv_heads; g.groups = g.H / g.Hkv;
  g.q_len = a->q_len; g.kv_len = a->kv_len; g.d_real = a->head_dim;
  g.elem = a->dtype;
  g.sm_scale = a->sm_scale;
  g.scale_log2 = (float)((double)a->sm_scale * 1.4426950408889634);
  g.ores = w->o_residual;
  sink_pattern(g, w);
  sink_fwd_plan(g);
  return g;
}

// bytes of the key ranges' parts: O [.., 16][D], then (m, l, n) [.., 16]
size_t sink_fwd_workspace(const SinkArgs& g) {
  if (g.splits <= 1) return 0;
  const size_t rows = (size_t)g.B * g.Hkv * g.row_tiles * g.splits * 16;
  return rows * ((g.d_real <= 64 ? 64 : 128) + 3) * sizeof(float);
}

esa_status sink_fwd_shape(const esa_fwd_args* a, const esa_window* w) {
  if (!a) return ESA_ERR_NULL;
  return sink_check(a->dtype, a->batch, a->num_heads, a->num_kv_heads, a->q_len, a->kv_len,
                    a->head_dim, a->sm_scale, w);
}

// Row stride of delta and lse2 (whole 16 bytes a head)
int sink_qpad(int q_len) { return (q_len + 3) / 4 * 4; }

// How the rows of a kv head's key blocks are cut, in stages of 64 rows and
// heads.  The chip runs `slots` blocks at a time (two a CU; float32 products
// leave a CU nothing for a second: 2 x 2048 rows, 8 heads of 64, window 256, 336
// blocks counted on 256 slots 76 us, on 512 100); a chunk costs what its stages
// do and about `part` stages more for its float32 part (written, read and
// joined; one where float32 products make a stage itself as long).  Counted so, with the blocks alike (a window):
//   a sinks' block is cut into pieces of a window block's size, or of its chunks';
//   of all blocks the whole rounds stay whole, and those that would run as an
//   unfilled last round are cut so that they fill it together (8192 rows, 8 kv
//   heads of 4 query heads, window 1024 and 4 sinks, head_dim 128: 568 blocks on
//   512 slots, two rounds of 72 stages against one and a fifth: 480 us and 365,
//   before the kernel itself was faster);
//   or all are cut, where that ends sooner (4096 rows, 32 heads on one kv head,
//   window 512: 32 blocks of 320 stages, backward 692 us whole, 205 cut);
// where the first blocks see many more rows than the last (a window near the
// sequence's length) all are cut alike, to at most 2/3 of a slot's share.
void sink_bwd_plan(SinkArgs& g) {
  g.nkb = (g.kv_len + 127) / 128;
  g.qpad = sink_qpad(g.q_len);
  const int64_t slots = g.elem == ESA_F32 ? 256 : 512, part = g.elem == ESA_F32 ? 1 : 6;
  const int64_t kv = (int64_t)g.B * g.Hkv;
  const int n_sink = std::min(g.nkb, (g.sinks + 127) / 128);
  auto stages = [&](int64_t rows) { return (rows + 63) / 64 * g.groups; };
  const int64_t one = stages(std::min<int64_t>(g.q_len, (int64_t)g.window + 127));
  // a block's rows are cut short by the sequence's end: the average of them
  const int64_t n_reg = g.nkb - n_sink;
  const int64_t span = std::min<int64_t>(g.window + 127, g.q_len);
  const double mean = 1.0 - 0.5 * (double)span / (double)std::max<int64_t>(g.q_len, 1);
  const bool alike = mean >= 0.75;
  int64_t cut = 1, n_last = 0, cut_last = 1;
  if (!alike && n_reg > 0) {
    const double share = (double)kv * n_reg * one * mean / (double)slots;
    cut = (int64_t)std::max(1.0, std::min(64.0, std::ceil(1.5 * one / share)));
    cut = std::max<int64_t>(1, std::min<int64_t>(cut, 4 * slots / (kv * n_reg)));
  }
  // the sinks' pieces as long as the others' chunks, within 256 MiB of parts
  auto sinks_cut = [&](int64_t piece) {
    if (n_sink == 0) return int64_t(1);
    const int64_t c = (stages(g.q_len) + piece - 1) / std::max<int64_t>(1, piece);
    return std::max<int64_t>(1, std::min<int64_t>({c, 128, 2048 / (kv * n_sink)}));
  };
  int64_t sink_cut = sinks_cut(std::max<int64_t>(1, one / cut));
  const int64_t total = kv * n_sink * sink_cut + kv * n_reg;
  if (alike && n_reg > 0 && total % slots != 0 && total < 8 * slots) {
    // the time, in stages, of `whole` blocks and then `chunks` chunks of `size`,
    // each taken by the next free slot
    auto time = [&](int64_t whole, int64_t chunks, int64_t size) {
      const int64_t rounds = whole / slots, rem = whole % slots;
      int64_t k = 0;  // chunks a slot that was free after `rounds`
      while ((slots - rem) * k + rem * std::max<int64_t>(0, (k * size - one) / size) < chunks) ++k;
      return std::max(rounds * one + k * size, (rounds + (rem > 0)) * one);
    };
    int64_t best = time(total, 0, one);
    const int64_t over = std::min<int64_t>(n_reg, (total % slots + kv - 1) / kv);
    for (int64_t c = 2; c <= 16 && c <= one; ++c) {
      const int64_t piece = (one + c - 1) / c;
      // the blocks past the whole rounds alone, then all of them and the sinks'
      if (kv * over * c <= 4 * slots) {
        const int64_t t = time(total - kv * over, kv * over * c, piece + part);
        if (t < best) {
          best = t;
          n_last = over;
          cut_last = c;
        }
      }
      if (kv * n_reg * c <= 4 * slots) {
        const int64_t cs = sinks_cut(piece);
        const int64_t size = std::max(piece, (stages(g.q_len) + cs - 1) / cs * (n_sink > 0));
        const int64_t t = time(0, kv * (n_sink * cs + n_reg * c), size + part);
        if (t < best) {
          best = t;
          n_last = n_reg;
          cut_last = c;
        }
      }
    }
    if (n_last == n_reg) sink_cut = sinks_cut((one + cut_last - 1) / cut_last);
  }
  g.cls_n[0] = n_sink;
  g.cls_cut[0] = (int)sink_cut;
  g.cls_n[1] = (int)(n_reg - n_last);
  g.cls_cut[1] = (int)cut;
  g.cls_n[2] = (int)n_last;
  g.cls_cut[2] = (int)cut_last;
}

struct SinkBwdSizes {
  size_t stat, part;  // bytes of delta (and of lse2), of the parts
  size_t total() const { return 2 * stat + part; }
};
SinkBwdSizes sink_bwd_sizes(const SinkArgs& g) {
  SinkBwdSizes z;
  z.stat = ((size_t)g.B * g.H * g.qpad * sizeof(float) + 255) / 256 * 256;
  size_t cut = 0;
  for (int c = 0; c < 3; ++c) cut += g.cls_cut[c] > 1 ? (size_t)g.cls_n[c] * g.cls_cut[c] : 0;
  z.part = (size_t)g.B * g.Hkv * cut * 2 * 128 * (g.d_real <= 64 ? 64 : 128) * sizeof(float);
  return z;
}

esa_status sink_bwd_shape(const esa_bwd_args* a, const esa_window* w) {
  if (!a) return ESA_ERR_NULL;
  return sink_check(a->dtype, a->batch, a->num_heads, a->num_kv_heads, a->q_len, a->kv_len,
                    a->head_dim, a->sm_scale, w);
}

SinkArgs sink_bwd_args(const esa_bwd_args* a, const esa_window* w) {
  SinkArgs g{};
  g.q = a->q; g.k = a->k; g.v = a->v; g.o = (void*)a->o; g.dout = a->dout;
  g.dq = a->dq; g.dk = a->dk; g.dv = a->dv; g.lse = (float*)a->lse;
  g.qsb = a->q_stride_b; g.qsh = a->q_stride_h; g.qss = a->q_stride_s;
  g.ksb = a->k_stride_b; g.ksh = a->k_stride_h; g.kss = a->k_stride_s;
  g.vsb = a->v_stride_b; g.vsh = a->v_stride_h; g.vss = a->v_stride_s;
  g.osb = a->o_stride_b; g.osh = a->o_stride_h; g.oss = a->o_stride_s;
  g.dosb = a->dout_stride_b; g.dosh = a->dout_stride_h; g.doss = a->dout_stride_s;
  g.dqsb = a->dq_stride_b; g.dqsh = a->dq_stride_h; g.dqss = a->dq_stride_s;
  g.dksb = a->dk_stride_b; g.dksh = a->dk_stride_h; g.dkss = a->dk_stride_s;
  g.dvsb = a->dv_stride_b; g.dvsh = a->dv_stride_h; g.dvss = a->dv_stride_s;
  g.lsb = a->lse_stride_b; g.lsh = a->lse_stride_h;
  g.B = a->batch; g.H = a->num_heads; g.Hkv = a->num_kv_heads; g.groups = g.H / g.Hkv;
  g.q_len = a->q_len; g.kv_len = a->kv_len; g.d_real = a->head_dim;
  g.elem = a->dtype;
  g.sm_scale = a->sm_scale;
  g.scale_log2 = (float)((double)a->sm_scale * 1.4426950408889634);
  g.ores = w->o_residual;
  sink_pattern(g, w);
  sink_bwd_plan(g);
  return g;
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

esa_status esa_sink_window_fwd_workspace_size(const esa_fwd_args* a, const esa_window* w,
                                              size_t* bytes) {
  if (!bytes) return ESA_ERR_NULL;
  const esa_status s = sink_fwd_shape(a, w);
  if (s != ESA_OK) return s;
  *bytes = a->batch == 0 || a->q_len == 0 ? 0 : sink_fwd_workspace(sink_fwd_args(a, w));
  return ESA_OK;
}

esa_status esa_sink_window_fwd(const esa_fwd_args* a, const esa_window* w, void* workspace,
                               size_t workspace_bytes, void* stream) {
  esa_status s = sink_fwd_shape(a, w);
  if (s != ESA_OK) return s;
  if (a->batch == 0 || a->q_len == 0) return ESA_OK;
  if (!a->q || !a->k || !a->v || !a->o) return ESA_ERR_NULL;
  const int es = a->dtype == ESA_F32 ? 4 : 2, epc = 16 / es;
  if (!stage_span_ok(a->k_stride_s, es) || !stage_span_ok(a->v_stride_s, es))
    return ESA_ERR_UNSUPPORTED;
  if ((s = sink_rows_ok(a->q, a->q_stride_b, a->q_stride_h, a->q_stride_s, epc)) != ESA_OK ||
      (s = sink_rows_ok(a->k, a->k_stride_b, a->k_stride_h, a->k_stride_s, epc)) != ESA_OK ||
      (s = sink_rows_ok(a->v, a->v_stride_b, a->v_stride_h, a->v_stride_s, epc)) != ESA_OK ||
      (s = sink_rows_ok(a->o, a->o_stride_b, a->o_stride_h, a->o_stride_s, epc)) != ESA_OK)
    return s;
  if (!aligned(w->o_residual, 16)) return ESA_ERR_ALIGN;
  SinkArgs g = sink_fwd_args(a, w);
  const size_t need = sink_fwd_workspace(g);
  if (need > 0) {
    if (!workspace) return ESA_ERR_NULL;
    if (!aligned(workspace, 16)) return ESA_ERR_ALIGN;
    if (workspace_bytes < need) return ESA_ERR_CAPACITY;
    g.partial = (float*)workspace;
    g.part_ml = g.partial + (size_t)g.B * g.Hkv * g.row_tiles * g.splits * 16 *
                                (g.d_real <= 64 ? 64 : 128);
  }
  const hipError_t e = g.decode ? launch_sink_decode(g, (hipStream_t)stream)
                                : launch_sink_fwd(g, (hipStream_t)stream);
  return e == hipSuccess ? ESA_OK : ESA_ERR_HIP;
}

esa_status esa_sink_window_bwd_workspace_size(const esa_bwd_args* a, const esa_window* w,
                                              size_t* bytes) {
  if (!bytes) return ESA_ERR_NULL;
  const esa_status s = sink_bwd_shape(a, w);
  if (s != ESA_OK) return s;
  *bytes = a->batch == 0 || a->q_len == 0 ? 0 : sink_bwd_sizes(sink_bwd_args(a, w)).total();
  return ESA_OK;
}

esa_status esa_sink_window_bwd(const esa_bwd_args* a, const esa_window* w, void* workspace,
                               size_t workspace_bytes, void* stream) {
  esa_status s = sink_bwd_shape(a, w);
  if (s != ESA_OK) return s;
  if (a->batch == 0 || a->q_len == 0) return ESA_OK;
  if (!a->q || !a->k || !a->v || !a->o || !a->dout || !a->dq || !a->dk || !a->dv || !a->lse)
    return ESA_ERR_NULL;
  const int es = a->dtype == ESA_F32 ? 4 : 2, epc = 16 / es;
  if (!stage_span_ok(a->k_stride_s, es) || !stage_span_ok(a->v_stride_s, es) ||
      !stage_span_ok(a->q_stride_s, es) || !stage_span_ok(a->dout_stride_s, es))
    return ESA_ERR_UNSUPPORTED;
  if ((s = sink_rows_ok(a->q, a->q_stride_b, a->q_stride_h, a->q_stride_s, epc)) != ESA_OK ||
      (s = sink_rows_ok(a->k, a->k_stride_b, a->k_stride_h, a->k_stride_s, epc)) != ESA_OK ||
      (s = sink_rows_ok(a->v, a->v_stride_b, a->v_stride_h, a->v_stride_s, epc)) != ESA_OK ||
      (s = sink_rows_ok(a->o, a->o_stride_b, a->o_stride_h, a->o_stride_s, epc)) != ESA_OK ||
      (s = sink_rows_ok(a->dout, a->dout_stride_b, a->dout_stride_h, a->dout_stride_s, epc)) != ESA_OK ||
      (s = sink_rows_ok(a->dq, a->dq_stride_b, a->dq_stride_h, a->dq_stride_s, epc)) != ESA_OK ||
      (s = sink_rows_ok(a->dk, a->dk_stride_b, a->dk_stride_h, a->dk_stride_s, epc)) != ESA_OK ||
      (s = sink_rows_ok(a->dv, a->dv_stride_b, a->dv_stride_h, a->dv_stride_s, epc)) != ESA_OK)
    return s;
  if (!aligned(w->o_residual, 16)) return ESA_ERR_ALIGN;
  SinkArgs g = sink_bwd_args(a, w);
  const SinkBwdSizes z = sink_bwd_sizes(g);
  if (!workspace) return ESA_ERR_NULL;
  if (!aligned(workspace, 16)) return ESA_ERR_ALIGN;
  if (workspace_bytes < z.total()) return ESA_ERR_CAPACITY;
  g.delta = (float*)workspace;
  g.lse2 = (float*)((char*)workspace + z.stat);
  g.partial = (float*)((char*)workspace + 2 * z.stat);
  return launch_sink_bwd(g, (hipStream_t)stream) == hipSuccess ? ESA_OK : ESA_ERR_HIP;
}

}  // extern "C"
