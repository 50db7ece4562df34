// Attention over a causal sliding window and a few first keys that stay
// visible (sinks), gfx950: what the forward, backward and decode kernels
// share.
//
// Row r of sequence b sits at position p = base(b) + r; its keys are
//   f <= j <= p  and  (p - j < window  or  j - f < sinks),   f = first_key(b).
// The kernels see the pattern as ranges: nothing but these numbers decides
// which key blocks a row block visits and which keys of a block count.
#pragma once
#include "esa_tile.hpp"

namespace esa {

struct SinkArgs {
  const void *q, *k, *v;
  void* o;
  float* lse;
  void* ores;  // what rounding o lost, in o's type and layout, or NULL
  const void* dout;
  void *dq, *dk, *dv;
  int64_t qsb, qsh, qss, ksb, ksh, kss, vsb, vsh, vss, osb, osh, oss, lsb, lsh;
  int64_t dosb, dosh, doss, dqsb, dqsh, dqss, dksb, dksh, dkss, dvsb, dvsh, dvss;
  int B, H, Hkv, groups, q_len, kv_len;
  int d_real;  // head_dim: dims d_real .. D - 1 of a kernel's D read as zeros
  int window, sinks;  // (both at most kv_len)
  const int64_t* pos;  // positions, or NULL (row r is position r)
  int64_t pos_sb;      // 0: shared by the batch
  const int64_t* first;  // first keys, or NULL (0)
  int elem;
  float sm_scale, scale_log2;
  int nqb;        // row blocks a head
  int xcd_runs;   // the grid's workgroups of one XCD take consecutive items
  // backward
  float* delta;  // [B, H, qpad] rowsum(dO * O)
  float* lse2;   // [B, H, qpad] log2(e) * lse
  int qpad;
  // a kv head's 128-key blocks in three classes, one after the other (the
  // sinks', the next, the last): their numbers and how many chunks the rows
  // of each class' blocks are cut into
  int nkb;
  int cls_n[3], cls_cut[3];
  float* partial;             // partial sums of the blocks with more than one chunk
  // Key ranges side by side (decode: of a (sequence, kv head, row tile); the
  // forward: of a row block), whose parts a join kernel adds up: row i of a kv
  // head's groups * q_len (row_of) leaves, for range s, O in partial[unit][D] and
  // (m, l, n) in part_ml[unit][3], unit = ((bkv row_tiles + i / 16) splits + s) 16
  // + i % 16
  bool decode;                // the decode kernel's row tiles, or the forward's blocks
  int splits;
  int row_tiles;              // 16-row tiles of a kv head's rows
  float* part_ml;
};

// Where a sequence's rows and keys start.  ok: the first position lies inside
// the cache.
struct SeqInfo {
  int base, first;
  bool ok;
};
__device__ __forceinline__ SeqInfo seq_info(const SinkArgs& A, int b) {
  SeqInfo s{0, 0, true};
  if (A.pos) {
    int64_t p = A.pos[(int64_t)b * A.pos_sb];
    p += p < 0 ? A.kv_len : 0;
    s.ok = p >= 0 && p < A.kv_len;
    s.base = s.ok ? (int)p : 0;
  }
  if (A.first) {
    const int64_t f = A.first[b];
    s.first = (int)(f < 0 ? 0 : f > A.kv_len ? A.kv_len : f);
  }
  return s;
}

// Row r's own position is base + r, inside the cache (else: a NaN row).
__device__ __forceinline__ bool row_valid(const SinkArgs& A, const SeqInfo& s, int b, int r) {
  if (!A.pos) return true;
  int64_t p = A.pos[(int64_t)b * A.pos_sb + r];
  p += p < 0 ? A.kv_len : 0;
  return s.ok && p == (int64_t)s.base + r && p < A.kv_len;
}

// The keys of [k0, k0 + 32) that the row at position p sees, as bits.
__device__ __forceinline__ uint32_t seen_keys(int p, int k0, int window, int sink_end) {
  const uint32_t win = range_word(p - window + 1 - k0, p - k0, 0);
  return win | range_word(0, min(sink_end - 1, p) - k0, 0);
}
// The rows (positions) of [p0, p0 + 32), up to p_last, that see key j, as bits.
__device__ __forceinline__ uint32_t seen_rows(int j, int p0, int p_last, int window,
                                              int sink_end) {
  const int hi = j < sink_end ? p_last : min(p_last, j + window - 1);
  return range_word(j - p0, hi - p0, 0);
}
// Rows [p0, p1] against keys [k0, k0 + 32): is every pair visible, is none?
__device__ __forceinline__ bool all_seen(int p0, int p1, int k0, int window, int sink_end) {
  return k0 + 31 <= p0 && (k0 > p1 - window || k0 + 32 <= sink_end);
}
__device__ __forceinline__ bool none_seen(int p0, int p1, int k0, int window, int sink_end) {
  return k0 > p1 || (k0 + 31 <= p0 - window && k0 >= sink_end);
}

// A row kernel's work item: a kv head's row blocks from the last (the most
// keys), the query heads that share it next to each other, so that an XCD
// works on the same keys at a time.
struct RowItem {
  int b, kvh, h, qb, split;
};
__device__ __forceinline__ RowItem row_item(const SinkArgs& A) {
  int item = blockIdx.x;
  if (A.xcd_runs) item = (item & 7) * ((int)gridDim.x >> 3) + (item >> 3);
  RowItem it;
  it.split = 0;
  if (A.splits > 1) {
    it.split = item % A.splits;
    item /= A.splits;
  }
  const int per = A.nqb * A.groups;
  const int bkv = item / per, rem = item - bkv * per;
  it.qb = A.nqb - 1 - rem / A.groups;
  it.b = bkv / A.Hkv;
  it.kvh = bkv - it.b * A.Hkv;
  it.h = it.kvh * A.groups + rem % A.groups;
  return it;
}
// Whole kv heads fall to each XCD (workgroup id % 8) where their number allows.
inline int sink_xcd_runs(const SinkArgs& a, int64_t grid) {
  return ((int64_t)a.B * a.Hkv) % 8 == 0 && grid % 8 == 0;
}

// The key stages (32 keys) of 128 rows from r0: n_sink stages of the sinks, then
// stages from m0 to the last row's position; one run where the two meet.
struct KeyStages {
  int f, n_sink, m0, n_all;
  int pb;  // the last row's position, inside the cache
  __device__ __forceinline__ int key0(int i) const {
    return i < n_sink ? f + i * 32 : m0 + (i - n_sink) * 32;
  }
};
// What the rows [p0, p0 + 31] of one wave (its last one p1, no row: p1 < p0)
// see of those stages, as ranges of their indices: none of a stage past `last`,
// or before `first` and the sinks; every pair of stages full_lo .. full_hi.
// (Sink stages count as partly seen.)
struct WaveStages {
  int last, first, sinks, full_lo, full_n;
  __device__ __forceinline__ bool sees(int i) const {
    return i <= last && (i >= first || i < sinks);
  }
  __device__ __forceinline__ bool full(int i) const { return (uint32_t)(i - full_lo) < (uint32_t)full_n; }
};
__device__ __forceinline__ WaveStages wave_stages(const KeyStages& k, int p0, int p1, int window,
                                                  int sink_end) {
  auto floor_div = [](int a) { return a >> 5; };
  WaveStages w;
  // k0 <= p1;  k0 + 31 > p0 - window;  k0 < sink_end
  w.last = p1 < p0 ? -1 : k.n_sink + max(floor_div(p1 - k.m0), -1);
  w.first = k.n_sink + floor_div(max(p0 - window + 1 - k.m0, 0));
  w.sinks = k.n_sink + (sink_end > k.m0 ? floor_div(sink_end - 1 - k.m0) + 1 : 0);
  // k0 > p0 + 31 - window and k0 + 31 <= p0
  w.full_lo = k.n_sink + max(floor_div(p0 + 31 - window - k.m0) + 1, 0);
  w.full_n = max(k.n_sink + floor_div(p0 + 1 - k.m0) - w.full_lo, 0);
  return w;
}
__device__ __forceinline__ KeyStages key_stages(const SinkArgs& A, const SeqInfo& si, int r0,
                                                int sink_end) {
  KeyStages k;
  k.f = si.first;
  k.pb = min(si.base + min(r0 + 127, A.q_len - 1), A.kv_len - 1);
  const int lo = max(k.f, si.base + r0 - A.window + 1);
  k.n_sink = lo > k.f && k.pb >= k.f ? (min(sink_end, lo) - k.f + 31) / 32 : 0;
  k.m0 = lo;
  if (k.n_sink > 0 && lo <= k.f + k.n_sink * 32) {
    k.n_sink = 0;
    k.m0 = k.f;
  }
  k.n_all = k.n_sink + (k.pb >= k.m0 ? (k.pb - k.m0) / 32 + 1 : 0);
  return k;
}

// ---------------------------------------------------------------------------
// Products of 32 x 32 blocks of one wave, for 16-bit types and float32.  Each
// lane owns column l % 32 (a row of q, or a key); hf = l / 32.
//   row_product   S[i][col] = sum_d X[i][d] col[d]: X's rows from LDS as the A
//                 operand, the lane's own row (Frag) as B
//   col_product   Y^T[d][col] += sum_i X[i][d] P[i][col]: the same LDS rows
//                 read by columns; P straight from a product's accumulators
// Accumulator register r of lane half hf is row 8 (r / 4) + 4 hf + r % 4.
// LDS rows are D elements unpadded, their 16-byte chunks XOR-swizzled by the
// row, so that both kinds of read meet each bank once.
// TIGHT: a kernel short of registers forms a read's address from one base with
// an exclusive or (the chunk's bits, which the swizzle and the read's place
// share) for each product anew, instead of keeping one register a read.
// DR: the dims that the products take (96 where a head has no more: LDS rows keep
// D's layout; 8192 rows, 32 heads on 8 of 96, window 1024, bf16: forward 152 us,
// backward 475, with 128 dims' products 179 and 541)
template <int D, Elem E, bool TIGHT = false, int DR = D>
struct SinkTile {
  using M = MmaT<E>;
  using V8 = typename M::v8;
  static constexpr int ES = 2;
  static constexpr int EPC = 8;        // elements of a chunk
  static constexpr int NS = DR / 16, ND = DR / 32;
  static constexpr int CPR = D / 8;    // chunks of a row
  struct Frag {
    V8 f[NS];
  };
  struct P {
    uint32_t w[8];
  };
  using LdsT = uint16_t;
  static constexpr uint32_t kOne = E == Elem::bf16 ? 0x3F80u : 0x3C00u;

  int ra[TIGHT ? 1 : NS];  // byte offsets of a 32-row block's row reads
  int ca[TIGHT ? 1 : ND];  // ... of its column reads, rows 4 hf + 0 .. 3 (+ 16 u)
  int hf;

  static __device__ __forceinline__ int swz(int row) { return swz_k<(D >= 128 ? 128 : 64)>(row); }
  __device__ __forceinline__ void init(int lane) {
    hf = lane >> 5;
    const int l32 = lane & 31, g4 = lane >> 4, lam = lane & 15;
#pragma unroll
    for (int s = 0; s < (TIGHT ? 1 : NS); ++s) ra[s] = 2 * (l32 * D + 8 * ((2 * s + hf) ^ swz(l32)));
    const int row = 4 * hf + (lam >> 2);
#pragma unroll
    for (int d = 0; d < (TIGHT ? 1 : ND); ++d) {
      const int col = 32 * d + 16 * (g4 & 1) + 4 * (lam & 3);
      ca[d] = 2 * (row * D + 8 * ((col >> 3) ^ swz(row)) + (col & 7));
    }
  }
  __device__ __forceinline__ void load_frag(Frag& f, const void* row, bool ok, int d_real) const {
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      u32x4 raw = {0u, 0u, 0u, 0u};
      const int d = 16 * s + 8 * hf;
      if (ok && d < d_real) raw = *(const u32x4*)((const uint16_t*)row + d);
      f.f[s] = __builtin_bit_cast(V8, raw);
    }
  }
  // c + the lane's share (its half of the dims) of the product of two rows
  static __device__ __forceinline__ float dot(const Frag& a, const Frag& b, float c) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        c = __builtin_fmaf(ElemT<E>::chunk(__builtin_bit_cast(u32x4, a.f[s]), e),
                           ElemT<E>::chunk(__builtin_bit_cast(u32x4, b.f[s]), e), c);
    return c;
  }
  __device__ __forceinline__ void row_product(f32x16& acc, const LdsT* buf, int rb,
                                              const Frag& f) const {
    V8 a[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) a[s] = row_operand(buf, rb, s);
#pragma unroll
    for (int s = 0; s < NS; ++s) acc = M::mfma32(a[s], f.f[s], acc);
  }
  // A base that the compiler takes for a new value (what a tight kernel's reads
  // of one product are formed from, so none is kept for the next)
  static __device__ __forceinline__ int fresh(int base) {
    if constexpr (TIGHT) asm volatile("" : "+v"(base));
    return base;
  }
  __device__ __forceinline__ V8 row_operand(const LdsT* buf, int rb, int s, int base) const {
    const int at = TIGHT ? base ^ (32 * s) : ra[s];
    return *(const V8*)((const char*)buf + at + 64 * rb * D);
  }
  __device__ __forceinline__ V8 row_operand(const LdsT* buf, int rb, int s) const {
    return row_operand(buf, rb, s, ra[0]);
  }
  // one product of col_product: rows 16 u .. of the block
  static __device__ __forceinline__ void col_step(f32x16& acc, const u32x4& a, const P& p, int u) {
    const u32x4 b = {p.w[4 * u], p.w[4 * u + 1], p.w[4 * u + 2], p.w[4 * u + 3]};
    acc = M::mfma32(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), acc);
  }
  __device__ __forceinline__ P pack(const f32x16& v) const {
    P p;
#pragma unroll
    for (int q = 0; q < 8; ++q) p.w[q] = M::pack2(v[2 * q], v[2 * q + 1]);
    return p;
  }
  // the A operand of dims 32 d .. and rows 16 u .. of block rb, by columns
  __device__ __forceinline__ u32x4 col_operand(const LdsT* buf, int rb, int d, int u) const {
    return col_operand(buf, rb, d, u, ca[0]);
  }
  __device__ __forceinline__ u32x4 col_operand(const LdsT* buf, int rb, int d, int u,
                                               int base) const {
    const int at = TIGHT ? base ^ (64 * d) : ca[d];
    const char* p1 = (const char*)buf + at + 2 * (32 * rb + 16 * u) * D;
    const char* p2 = (const char*)buf + (at ^ 32) + 2 * (32 * rb + 16 * u + 8) * D;
    const s16x4 v[2] = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p1),
                        __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p2)};
    return __builtin_bit_cast(u32x4, v);
  }
  __device__ __forceinline__ void col_product(f32x16 (&acc)[ND], const LdsT* buf, int rb,
                                              const P& p) const {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const u32x4 a = col_operand(buf, rb, d, u);
        const u32x4 b = {p.w[4 * u], p.w[4 * u + 1], p.w[4 * u + 2], p.w[4 * u + 3]};
        acc[d] = M::mfma32(__builtin_bit_cast(V8, a), __builtin_bit_cast(V8, b), acc[d]);
      }
  }
  // dims 32 d + 8 q4 + 4 hf .. of the lane's own row
  static __device__ __forceinline__ void store4(void* row, int dim, float a, float b, float c,
                                                float e) {
    typename M::v4 v;
    v[0] = (typename M::s)a;
    v[1] = (typename M::s)b;
    v[2] = (typename M::s)c;
    v[3] = (typename M::s)e;
    *(typename M::v4*)((uint16_t*)row + dim) = v;
  }
  // scale * x, one 32-dim block of an accumulator, to dims dim0 .. of the lane's
  // row: the row's two lanes trade halves and store 16 bytes each (with 8 a lane
  // the stores of 128 rows took as long as three stages)
  static __device__ __forceinline__ void store32(void* row, int dim0, const f32x16& x, float scale,
                                                 int hf, int d_real, bool in) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        w[q] = M::pack2(x[8 * j + 2 * q] * scale, x[8 * j + 2 * q + 1] * scale);
      const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
      const auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
      const int dim = dim0 + 16 * j + 8 * hf;
      if (in && dim < d_real)
        *(u32x4*)((uint16_t*)row + dim) = u32x4{a[0], b[0], a[1], b[1]};
    }
  }
  static __device__ __forceinline__ float rounded(float x) { return (float)(typename M::s)x; }
  static __device__ __forceinline__ float psum(const P& p, float c) {
#pragma unroll
    for (int q = 0; q < 8; ++q) c = M::dot2(p.w[q], c);
    return c;
  }
};

template <int D, bool TIGHT, int DR>
struct SinkTile<D, Elem::f32, TIGHT, DR> {
  static constexpr int ES = 4;
  static constexpr int EPC = 4;
  static constexpr int NU = DR / 8, ND = DR / 32;
  static constexpr int CPR = D / 4;
  struct Frag {
    f32x4 f[NU];
  };
  using P = f32x16;
  using LdsT = float;

  int ra;     // row reads: the lane's row; chunk 2 u + hf is XORed in below
  int sw;
  int ca[4];  // column reads of rows 4 hf + t
  int hf;

  static __device__ __forceinline__ int swz(int row) { return row & 7; }
  __device__ __forceinline__ void init(int lane) {
    hf = lane >> 5;
    const int l32 = lane & 31;
    ra = l32 * D;
    sw = l32 & 7;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int row = 4 * hf + t;
      ca[t] = row * D + 4 * ((l32 >> 2) ^ row) + (l32 & 3);
    }
  }
  __device__ __forceinline__ void load_frag(Frag& f, const void* row, bool ok, int d_real) const {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      f32x4 raw = {0.f, 0.f, 0.f, 0.f};
      const int d = 8 * u + 4 * hf;
      if (ok && d < d_real) raw = *(const f32x4*)((const float*)row + d);
      f.f[u] = raw;
    }
  }
  static __device__ __forceinline__ float dot(const Frag& a, const Frag& b, float c) {
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int t = 0; t < 4; ++t) c = __builtin_fmaf(a.f[u][t], b.f[u][t], c);
    return c;
  }
  __device__ __forceinline__ void row_product(f32x16& acc, const float* buf, int rb,
                                              const Frag& f) const {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const f32x4 a = *(const f32x4*)(buf + ra + 32 * rb * D + 4 * ((2 * u + hf) ^ sw));
#pragma unroll
      for (int t = 0; t < 4; ++t)
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[t], f.f[u][t], acc, 0, 0, 0);
    }
  }
  __device__ __forceinline__ P pack(const f32x16& v) const { return v; }
  __device__ __forceinline__ float col_operand(const float* buf, int rb, int d, int r) const {
    return buf[ca[r & 3] + (32 * rb + 8 * (r >> 2)) * D + 32 * d];
  }
  __device__ __forceinline__ void col_product(f32x16 (&acc)[ND], const float* buf, int rb,
                                              const P& p) const {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(col_operand(buf, rb, d, r), p[r], acc[d], 0,
                                                      0, 0);
  }
  static __device__ __forceinline__ void store4(void* row, int dim, float a, float b, float c,
                                                float e) {
    *(f32x4*)((float*)row + dim) = f32x4{a, b, c, e};
  }
  static __device__ __forceinline__ void store32(void* row, int dim0, const f32x16& x, float scale,
                                                 int hf, int d_real, bool in) {
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int dim = dim0 + 8 * q4 + 4 * hf;
      if (in && dim < d_real)
        store4(row, dim, x[4 * q4] * scale, x[4 * q4 + 1] * scale, x[4 * q4 + 2] * scale,
               x[4 * q4 + 3] * scale);
    }
  }
  static __device__ __forceinline__ float rounded(float x) { return x; }
  static __device__ __forceinline__ float psum(const P& p, float c) {
#pragma unroll
    for (int q = 0; q < 16; ++q) c += p[q];
    return c;
  }
};

// ROWS rows of D elements from one matrix into LDS, 16 bytes a lane and load.
// The buffer resource starts at a row of the matrix (`org`) and ends with its
// last one; a stage is reached by the scalar offset of its first row, and past
// 1 GiB from org the resource moves on, so offsets stay small however long the
// tensor is.  Whatever lies past the last row, or past head_dim, reads as zero.
// (A resource formed anew for every stage cost more scalar instructions than
// the stage's products have vector ones, and a third of the forward's time.)
template <int D, Elem E, int ROWS, int THREADS>
struct SinkStage {
  using T = SinkTile<D, E>;
  static constexpr int LOADS = ROWS * T::CPR / THREADS;
  static constexpr int BYTES = ROWS * D * T::ES;
  // rows of one round of loads: a multiple of the swizzle's period, so a lane's
  // rounds differ by a scalar alone
  static constexpr int ROUND = THREADS / T::CPR;
  static_assert(LOADS >= 1 && LOADS * THREADS == ROWS * T::CPR, "whole stage per load round");
  int off;
  __amdgpu_buffer_rsrc_t rs;
  const char* base;
  int64_t stride;  // bytes
  int rows;        // rows of the matrix
  int row_bytes;
  int org, reach;  // the resource's first row, and how many rows it serves

  __device__ __forceinline__ void init(const void* p, int64_t stride_elems, int n_rows, int d_real,
                                       int tid) {
    base = (const char*)p;
    stride = stride_elems * T::ES;
    rows = n_rows;
    row_bytes = d_real * T::ES;
    org = 0;
    reach = 0;
    const int row = tid / T::CPR, chunk = (tid % T::CPR) ^ T::swz(row);
    off = 16 * chunk < row_bytes ? (int)(row * stride) + 16 * chunk : 0x7ffffff0;
    // (0x7ffffff0 plus a stage's offset, below 2^30, is past every resource as
    // an unsigned number)
  }
  // another matrix of the same shape
  __device__ __forceinline__ void rebase(const void* p) {
    base = (const char*)p;
    reach = 0;
  }
  __device__ __forceinline__ void move(int row0) {
    const int64_t left = (int64_t)(rows - row0 - 1) * stride + row_bytes;
    const int n = rows > row0 ? (int)(left < 0x7fffff00 ? left : 0x7fffff00) : 0;
    rs = __builtin_amdgcn_make_buffer_rsrc((void*)(base + (int64_t)row0 * stride), (short)0, n,
                                           0x00020000);
    org = row0;
    reach = (int)((1u << 30) / (uint32_t)(stride > 16 ? stride : 16));
  }
  // rows row0 .. row0 + ROWS - 1 -> dst
  __device__ __forceinline__ void issue(int row0, void* dst, int wave) {
    if ((uint32_t)(row0 - org) >= (uint32_t)reach) move(row0);
    const int soff = (row0 - org) * (int)stride;
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
      load_lds16(rs, (uint16_t*)dst + (wave + j * (THREADS / 64)) * 512, off,
                 soff + j * ROUND * (int)stride);
  }
};

// Waits for this wave's loads into LDS, then for the other waves' (and for
// their reads of the buffer that is filled next).
__device__ __forceinline__ void stage_ready() {
  __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
  __syncthreads();
}

// Waits until at most LATER of this wave's loads are on their way, then for
// the other waves.
template <int LATER>
__device__ __forceinline__ void stage_wait() {
  static_assert(LATER < 64, "vmcnt counts to 63");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LATER) : "memory");
}

// Non-finite values.  A staged block also holds rows that a column does not
// see; they meet P = 0 in the products, and 0 * Inf is NaN (so is the mask's
// -inf plus an Inf score).  The kernels therefore look at what they stored:
// a row (or key) whose values came out non-finite is computed again from the
// pairs that it sees alone, by one wave in float32, so a hidden Inf or NaN
// reaches nothing and a visible one exactly what the formula gives.
//
// The keys of one row in order: n_sink sinks from f, then lo .. p.
struct RowKeys {
  int f, n_sink, lo, n;
  __device__ __forceinline__ int key(int i) const { return i < n_sink ? f + i : lo + i - n_sink; }
};
__device__ __forceinline__ RowKeys row_keys(int p, int f, int window, int sink_end) {
  RowKeys k;
  k.f = f;
  k.lo = max(f, p - window + 1);
  k.n_sink = max(0, min(sink_end, k.lo) - f);
  k.n = p < f ? 0 : k.n_sink + p - k.lo + 1;
  return k;
}

// sum_d a[d] b[d] over d_real elements (whole 16-byte chunks)
template <Elem E>
__device__ __forceinline__ float row_dot(const void* a, const void* b, int d_real) {
  using T = ElemT<E>;
  float s = 0.f;
#pragma unroll 1
  for (int d = 0; d < d_real; d += T::kPerChunk) {
    const u32x4 x = *(const u32x4*)((const typename T::T*)a + d);
    const u32x4 y = *(const u32x4*)((const typename T::T*)b + d);
#pragma unroll
    for (int e = 0; e < T::kPerChunk; ++e) s = __builtin_fmaf(T::chunk(x, e), T::chunk(y, e), s);
  }
  return s;
}

// Four dims of an output row, and (where the caller keeps it for a backward)
// what rounding them lost.
template <int D, Elem E>
__device__ __forceinline__ void store_out4(const SinkArgs& A, int64_t row, int dim, float a,
                                           float b, float c, float d) {
  using T = SinkTile<D, E>;
  T::store4((char*)A.o + row * T::ES, dim, a, b, c, d);
  if (A.ores)
    T::store4((char*)A.ores + row * T::ES, dim, a - T::rounded(a), b - T::rounded(b),
              c - T::rounded(c), d - T::rounded(d));
}

// The same of a 32-dim block of accumulators.
template <int D, Elem E>
__device__ __forceinline__ void store_out32(const SinkArgs& A, int64_t row, int dim0, f32x16 x,
                                            float scale, int hf, bool in) {
  using T = SinkTile<D, E>;
  T::store32((char*)A.o + row * T::ES, dim0, x, scale, hf, A.d_real, in);
  if (A.ores) {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = x[e] * scale - T::rounded(x[e] * scale);
    T::store32((char*)A.ores + row * T::ES, dim0, x, 1.f, hf, A.d_real, in);
  }
}

// Row `row` of one head from its own keys, by one wave: lanes take 64 keys at a
// time for the scores and the head's dims for the weighted sum.
template <Elem E>
__device__ void fix_row(const SinkArgs& A, int b, int h, int kvh, int row, int p, int f,
                        int sink_end, int lane) {
  using T = ElemT<E>;
  using EL = typename T::T;
  const EL* q = (const EL*)A.q + (int64_t)b * A.qsb + (int64_t)h * A.qsh + (int64_t)row * A.qss;
  const EL* k = (const EL*)A.k + (int64_t)b * A.ksb + (int64_t)kvh * A.ksh;
  const EL* v = (const EL*)A.v + (int64_t)b * A.vsb + (int64_t)kvh * A.vsh;
  const RowKeys rk = row_keys(p, f, A.window, sink_end);
  float m = -INFINITY, l = 0.f, acc[2] = {0.f, 0.f};
#pragma unroll 1
  for (int i0 = 0; i0 < rk.n; i0 += 64) {
    const bool in = i0 + lane < rk.n;
    float s = -INFINITY;
    if (in)
      s = row_dot<E>(q, k + (int64_t)rk.key(i0 + lane) * A.kss, A.d_real) * A.scale_log2;
    const float top = fmaxf(m, wave_max(s)), use = top == -INFINITY ? 0.f : top;
    const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - use);
    const float pr = in ? __builtin_amdgcn_exp2f(s - use) : 0.f;
    m = top;
    l = l * alpha + wave_sum(pr);
    acc[0] *= alpha;
    acc[1] *= alpha;
    const int n = min(64, rk.n - i0);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const float w = __shfl(pr, i, 64);
      const EL* vr = v + (int64_t)rk.key(i0 + i) * A.vss;
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (lane + 64 * c < A.d_real)
          acc[c] = __builtin_fmaf(w, T::load(vr + lane + 64 * c), acc[c]);
    }
  }
  const bool empty = rk.n <= 0;
  const int64_t at = (int64_t)b * A.osb + (int64_t)h * A.osh + (int64_t)row * A.oss;
#pragma unroll
  for (int c = 0; c < 2; ++c)
    if (lane + 64 * c < A.d_real) {
      const float y = empty ? 0.f : acc[c] / l;
      EL* o = (EL*)A.o + at + lane + 64 * c;
      T::store(o, y);
      if (A.ores) T::store((EL*)A.ores + at + lane + 64 * c, y - T::load(o));
    }
  if (A.lse && lane == 0)
    A.lse[(int64_t)b * A.lsb + (int64_t)h * A.lsh + row] =
        empty ? -INFINITY : (m + __log2f(l)) * 0.69314718055994530942f;
}

hipError_t launch_sink_fwd(const SinkArgs& a, hipStream_t stream);
hipError_t launch_sink_bwd(const SinkArgs& a, hipStream_t stream);
hipError_t launch_sink_decode(const SinkArgs& a, hipStream_t stream);
hipError_t launch_sink_rows_join(const SinkArgs& a, hipStream_t stream);

}  // namespace esa
