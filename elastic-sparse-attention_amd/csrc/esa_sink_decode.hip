// Decode form of attention over a causal window with sinks (gfx950): few rows
// per sequence against a long cache.
//
// The query heads that share a kv head (and the rows of a step) form tiles of
// 16 rows, so each key is read once for all of them; a tile's visible keys
// (the sinks, then the window) are cut into `splits` ranges, one workgroup
// each, and a range's keys go to its four waves 32 at a time.  A wave is on its
// own until the end: K rows straight into the registers that S^T = K Q^T
// takes, V rows into its part of LDS without registers, read back by columns
// for O^T += V^T P^T.  Then the waves' maxima, sums and O join in LDS and, if
// the keys were cut, the ranges' in a second kernel.
//
// Bound: HBM (every visible key and value is read once); what hides its
// latency is the number of waves, each with 32 keys' K and V in flight: 64
// sequences over 4096-key windows of 8 kv heads at head_dim 128, 1.08 GB, in
// 184 us (5.9 TB/s, the rate of a gather of such rows); 4 sequences over
// 131072 keys of 2 kv heads, 488 MB, in 94 us with the join.  One sequence is
// bound by latency: 1028 keys of 8 kv heads in 72 workgroups take 6.9 us and
// 3.4 the join (one workgroup of 16 waves a kv head and no join took 16.7: a
// CU alone draws 16 bytes a clock from HBM).
#include "esa_sink.hpp"

namespace esa {

namespace {

// Products of 32 keys and 16 rows (v_mfma_f32_16x16x32 and, float32, 16x16x4):
// lane l holds row l % 16; accumulator register r of tile t is key
// 16 t + 4 (l / 16) + r (S^T), or dim 16 t + 4 (l / 16) + r (O^T).
template <int D, Elem E>
struct DecodeTile {
  using M = MmaT<E>;
  using V8 = typename M::v8;
  using LdsT = uint16_t;
  static constexpr int ES = 2, EPC = 8, NK = D / 32, NO = D / 16, CPR = D / 8;
  struct Frag {
    u32x4 f[NK];
  };
  static __device__ __forceinline__ int swz(int row) { return swz_k<(D >= 128 ? 128 : 64)>(row); }
  // the 16-byte pieces of one row (of K or Q) this lane holds
  static __device__ __forceinline__ void load(Frag& f, const void* row, bool ok, int d_real, int g) {
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      f.f[s] = u32x4{0u, 0u, 0u, 0u};
      const int d = 32 * s + 8 * g;
      if (ok && d < d_real) f.f[s] = *(const u32x4*)((const uint16_t*)row + d);
    }
  }
  static __device__ __forceinline__ f32x4 scores(const Frag& k, const Frag& q) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NK; ++i)
      s = M::mfma16(__builtin_bit_cast(V8, k.f[i]), __builtin_bit_cast(V8, q.f[i]), s);
    return s;
  }
  // O^T += V^T P^T; returns the sum of P as the product used it
  static __device__ __forceinline__ float values(f32x4 (&o)[NO], const LdsT* v, const f32x4& p0,
                                                 const f32x4& p1, int lane) {
    const u32x4 pw = {M::pack2(p0[0], p0[1]), M::pack2(p0[2], p0[3]), M::pack2(p1[0], p1[1]),
                      M::pack2(p1[2], p1[3])};
    const int g = lane >> 4, lam = lane & 15;
    const int row = 4 * g + (lam >> 2);
#pragma unroll
    for (int d = 0; d < NO; ++d) {
      const int col = 16 * d + 4 * (lam & 3);
      const LdsT* a = v + row * D + 8 * ((col >> 3) ^ swz(row)) + (col & 7);
      const s16x4 x[2] = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)a),
                          __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(a + 16 * D))};
      o[d] = M::mfma16(__builtin_bit_cast(V8, x), __builtin_bit_cast(V8, pw), o[d]);
    }
    return M::dot2(pw[0], M::dot2(pw[1], M::dot2(pw[2], M::dot2(pw[3], 0.f))));
  }
};

template <int D>
struct DecodeTile<D, Elem::f32> {
  using LdsT = float;
  static constexpr int ES = 4, EPC = 4, NK = D / 16, NO = D / 16, CPR = D / 4;
  struct Frag {
    f32x4 f[NK];
  };
  static __device__ __forceinline__ int swz(int row) { return row & 7; }
  static __device__ __forceinline__ void load(Frag& f, const void* row, bool ok, int d_real, int g) {
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      f.f[s] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int d = 16 * s + 4 * g;
      if (ok && d < d_real) f.f[s] = *(const f32x4*)((const float*)row + d);
    }
  }
  static __device__ __forceinline__ f32x4 scores(const Frag& k, const Frag& q) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NK; ++i)
#pragma unroll
      for (int t = 0; t < 4; ++t)
        s = __builtin_amdgcn_mfma_f32_16x16x4f32(k.f[i][t], q.f[i][t], s, 0, 0, 0);
    return s;
  }
  static __device__ __forceinline__ float values(f32x4 (&o)[NO], const LdsT* v, const f32x4& p0,
                                                 const f32x4& p1, int lane) {
    const int g = lane >> 4, lam = lane & 15;
#pragma unroll
    for (int d = 0; d < NO; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 4 * g + r;  // (and row + 16, with the same swizzle)
        const LdsT* a = v + row * D + 4 * ((4 * d + (lam >> 2)) ^ swz(row)) + (lam & 3);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[0], p0[r], o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[16 * D], p1[r], o[d], 0, 0, 0);
      }
    return ((p0[0] + p0[1]) + (p0[2] + p0[3])) + ((p1[0] + p1[1]) + (p1[2] + p1[3]));
  }
};

typedef const __attribute__((address_space(1))) void global_cvoid;

// Row index -> its head and its place in the sequence
struct DecodeRow {
  int h, s;
};
__device__ __forceinline__ DecodeRow decode_row(const SinkArgs& A, int kvh, int i) {
  DecodeRow r;
  r.s = i / A.groups;
  r.h = kvh * A.groups + i - r.s * A.groups;
  return r;
}

// Final row: O and lse from the joined sums; by the lanes that hold its dims
__device__ __forceinline__ float decode_lse(float m, float l, bool empty) {
  return empty ? -INFINITY : (m + __log2f(l)) * 0.69314718055994530942f;
}

template <int D, Elem E>
__global__ __launch_bounds__(256, 2) void sink_decode_kernel(SinkArgs A) {
  using T = DecodeTile<D, E>;
  using LdsT = typename T::LdsT;
  using EL = typename ElemT<E>::T;
  constexpr int WAVES = 4, KEYS = 32;
  constexpr int VLOADS = KEYS * T::CPR / 64;
  // each wave's V rows; at the end, in the same place, every wave's O [16][D]
  constexpr int VBYTES = KEYS * D * T::ES, OSTRIDE = D + 4, OBYTES = 16 * OSTRIDE * 4;
  constexpr int BYTES = WAVES * (VBYTES > OBYTES ? VBYTES : OBYTES);
  __shared__ __attribute__((aligned(1024))) char smem[BYTES];
  __shared__ float mlbuf[WAVES][3][16];
  float(*obuf)[16 * OSTRIDE] = (float(*)[16 * OSTRIDE])smem;

  const int units = A.row_tiles * A.splits;
  const int bkv = blockIdx.x / units, u = blockIdx.x - bkv * units;
  const int rt = u / A.splits, split = u - rt * A.splits;
  const int b = bkv / A.Hkv, kvh = bkv - b * A.Hkv;
  const SeqInfo si = seq_info(A, b);
  const int f = si.first, sink_end = min(f + A.sinks, A.kv_len), W = A.window;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, lam = lane & 15;
  const int n_rows = A.groups * A.q_len;
  const int i_row = rt * 16 + lam;
  const bool row_in = i_row < n_rows;
  const DecodeRow row = decode_row(A, kvh, min(i_row, n_rows - 1));
  const int p = si.base + row.s;

  // ---- the tile's keys in order: sinks, then lo .. pb; this range's share
  const int pa = si.base + decode_row(A, kvh, rt * 16).s;
  const int pb = min(si.base + decode_row(A, kvh, min(rt * 16 + 15, n_rows - 1)).s, A.kv_len - 1);
  RowKeys rk;
  rk.f = f;
  rk.lo = max(f, pa - W + 1);
  rk.n_sink = pb >= f ? max(0, min(sink_end, rk.lo) - f) : 0;
  rk.n = rk.n_sink + max(0, pb - rk.lo + 1);
  // in whole 32-key pieces
  const int pieces = (rk.n + KEYS - 1) / KEYS;
  const int i0 = (int)((int64_t)pieces * split / A.splits) * KEYS;
  const int i1 = min((int)((int64_t)pieces * (split + 1) / A.splits) * KEYS, rk.n);

  const EL* kbase = (const EL*)A.k + (int64_t)b * A.ksb + (int64_t)kvh * A.ksh;
  const EL* vbase = (const EL*)A.v + (int64_t)b * A.vsb + (int64_t)kvh * A.vsh;
  typename T::Frag qf;
  T::load(qf, (const EL*)A.q + (int64_t)b * A.qsb + (int64_t)row.h * A.qsh +
                  (int64_t)row.s * A.qss, row_in, A.d_real, g);
  f32x4 o[T::NO];
#pragma unroll
  for (int d = 0; d < T::NO; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f, n_sum = 0.f;

  LdsT* const vmine = (LdsT*)(smem + wave * VBYTES);
  for (int i = i0 + wave * KEYS; i < i1; i += WAVES * KEYS) {
    // V: rows i .. i + 31 (past the end the last key's again, with P = 0; dims
    // past head_dim hold whatever, and are not stored)
#pragma unroll
    for (int j = 0; j < VLOADS; ++j) {
      const int slot = j * 64 + lane, r = slot / T::CPR;
      int chunk = (slot % T::CPR) ^ T::swz(r);
      chunk = chunk * T::EPC < A.d_real ? chunk : 0;
      const EL* src = vbase + (int64_t)rk.key(min(i + r, i1 - 1)) * A.vss + chunk * T::EPC;
      __builtin_amdgcn_global_load_lds((global_cvoid*)src, (lds_void*)((char*)vmine + j * 1024),
                                       16, 0, 0);
    }
    typename T::Frag k0, k1;
    T::load(k0, kbase + (int64_t)rk.key(min(i + lam, i1 - 1)) * A.kss, true, A.d_real, g);
    T::load(k1, kbase + (int64_t)rk.key(min(i + 16 + lam, i1 - 1)) * A.kss, true, A.d_real, g);
    f32x4 s0 = T::scores(k0, qf), s1 = T::scores(k1, qf);
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int ia = i + 4 * g + r, ib = ia + 16;
      const int ja = rk.key(ia), jb = rk.key(ib);
      const bool sa = ia < i1 && ja <= p && (p - ja < W || ja < sink_end);
      const bool sb = ib < i1 && jb <= p && (p - jb < W || jb < sink_end);
      s0[r] = sa ? s0[r] * A.scale_log2 : -INFINITY;
      s1[r] = sb ? s1[r] * A.scale_log2 : -INFINITY;
      top = fmaxf(top, fmaxf(s0[r], s1[r]));
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float m_new = fmaxf(m, top), use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - use);
    m = m_new;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s0[r] = __builtin_amdgcn_exp2f(s0[r] - use);
      s1[r] = __builtin_amdgcn_exp2f(s1[r] - use);
    }
    l = l * alpha + (((s0[0] + s0[1]) + (s0[2] + s0[3])) + ((s1[0] + s1[1]) + (s1[2] + s1[3])));
#pragma unroll
    for (int d = 0; d < T::NO; ++d) o[d] *= alpha;
    __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
    asm volatile("" ::: "memory");
    n_sum = n_sum * alpha + T::values(o, vmine, s0, s1, lane);
    // (this wave's reads of its V rows end before they are written again)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }

  // ---- the waves' results joined
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  n_sum += __shfl_xor(n_sum, 16, 64);
  n_sum += __shfl_xor(n_sum, 32, 64);
  __syncthreads();  // every wave is done with its V rows
#pragma unroll
  for (int d = 0; d < T::NO; ++d)
    *(f32x4*)(obuf[wave] + lam * OSTRIDE + 16 * d + 4 * g) = o[d];
  if (g == 0) {
    mlbuf[wave][0][lam] = m;
    mlbuf[wave][1][lam] = l;
    mlbuf[wave][2][lam] = n_sum;
  }
  __syncthreads();
  // 16 lanes a row: 4 dims each and pass
  const int jr = tid >> 4, c16 = tid & 15;
  const int ir = rt * 16 + jr;
  const bool jin = ir < n_rows;
  float mt = -INFINITY;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) mt = fmaxf(mt, mlbuf[w][0][jr]);
  const float mu = mt == -INFINITY ? 0.f : mt;
  float wgt[WAVES], lt = 0.f, nt = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    wgt[w] = mlbuf[w][0][jr] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mlbuf[w][0][jr] - mu);
    // (a wave without a key of the row: nothing, whatever its sums hold)
    if (wgt[w] != 0.f) {
      lt += wgt[w] * mlbuf[w][1][jr];
      nt += wgt[w] * mlbuf[w][2][jr];
    }
    if (mlbuf[w][1][jr] != mlbuf[w][1][jr]) lt = nt = __builtin_nanf("");
  }
  const DecodeRow jrow = decode_row(A, kvh, min(ir, n_rows - 1));
  const int pj = si.base + jrow.s;
  const bool whole = A.splits == 1;
  const float inv = whole ? (pj < f ? 0.f : 1.f / nt) : 1.f;
  const bool valid = jin && (!whole || row_valid(A, si, b, jrow.s));
  const int64_t orow = (int64_t)b * A.osb + (int64_t)jrow.h * A.osh + (int64_t)jrow.s * A.oss;
  const int64_t unit = (int64_t)blockIdx.x * 16 + jr;
  bool finite = true;
#pragma unroll
  for (int d0 = 0; d0 < D; d0 += 64) {
    const int dim = d0 + 4 * c16;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      y += wgt[w] * *(const f32x4*)(obuf[w] + jr * OSTRIDE + dim);
    if (dim < A.d_real)
      finite &= __builtin_isfinite((y[0] + y[1]) + (y[2] + y[3]));
    if (!jin || dim >= A.d_real) continue;
    if (whole) {
      if (!valid) y = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
      store_out4<D, E>(A, orow, dim, y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
    } else {
      *(f32x4*)(A.partial + unit * D + dim) = y;
    }
  }
  if (jin && c16 == 0) {
    if (whole) {
      if (A.lse)
        A.lse[(int64_t)b * A.lsb + (int64_t)jrow.h * A.lsh + jrow.s] =
            valid ? decode_lse(mt, lt, pj < f) : __builtin_nanf("");
    } else {
      float* ml = A.part_ml + unit * 3;
      ml[0] = mt;
      ml[1] = lt;
      ml[2] = nt;
    }
  }
  if (!whole) return;
  // rows that met a non-finite value, again from their own keys
  const bool met = valid && !(finite && __builtin_isfinite(lt));
  uint64_t bad = __builtin_amdgcn_ballot_w64(met);
  if (bad) __builtin_amdgcn_s_waitcnt(0);
#pragma unroll 1
  for (int q = 0; q < 4; ++q) {
    if (((bad >> (16 * q)) & 0xffffull) == 0) continue;
    const DecodeRow fr = decode_row(A, kvh, rt * 16 + wave * 4 + q);
    fix_row<E>(A, b, fr.h, kvh, fr.s, si.base + fr.s, f, sink_end, lane);
  }
}

// The key ranges of one row, joined in order: GR groups of lanes take every
// GR-th range, each lane 4 dims, then the groups' sums in LDS.
template <int D, Elem E>
__global__ __launch_bounds__(512) void sink_ranges_join_kernel(SinkArgs A) {
  constexpr int LPR = D / 4, GR = 512 / LPR;
  __shared__ __attribute__((aligned(16))) float ob[GR][D];
  __shared__ float wsum[GR][2];
  const int n_rows = A.groups * A.q_len;
  const int bkv = blockIdx.x / n_rows, ir = blockIdx.x - bkv * n_rows;
  const int b = bkv / A.Hkv, kvh = bkv - b * A.Hkv;
  const int rt = ir >> 4, jr = ir & 15;
  const DecodeRow row = decode_row(A, kvh, ir);
  const SeqInfo si = seq_info(A, b);
  const int f = si.first, sink_end = min(f + A.sinks, A.kv_len), p = si.base + row.s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t u0 = ((int64_t)bkv * A.row_tiles + rt) * A.splits;
  auto unit = [&](int s) { return (u0 + s) * 16 + jr; };
  // the maximum over all ranges: every wave by itself
  float mt = -INFINITY;
  for (int s = lane; s < A.splits; s += 64) mt = fmaxf(mt, A.part_ml[unit(s) * 3]);
  mt = wave_max(mt);
  const float mu = mt == -INFINITY ? 0.f : mt;
  const int gr = tid / LPR, dim = 4 * (tid % LPR);
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  float lt = 0.f, nt = 0.f;
  for (int s = gr; s < A.splits; s += GR) {
    const float* ml = A.part_ml + unit(s) * 3;
    const float ms = ml[0];
    const float w = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - mu);
    if (w != 0.f || ml[1] != ml[1]) {
      lt += w * ml[1];
      nt += w * ml[2];
    }
    if (dim < A.d_real) y += w * *(const f32x4*)(A.partial + unit(s) * D + dim);
  }
  *(f32x4*)(ob[gr] + dim) = y;
  if (dim == 0) {
    wsum[gr][0] = lt;
    wsum[gr][1] = nt;
  }
  __syncthreads();
  if (tid >= 64) return;
  lt = nt = 0.f;
  for (int q = 0; q < GR; ++q) {
    lt += wsum[q][0];
    nt += wsum[q][1];
  }
  const bool valid = row_valid(A, si, b, row.s);
  const float inv = !valid ? __builtin_nanf("") : p < f ? 0.f : 1.f / nt;
  const int64_t orow = (int64_t)b * A.osb + (int64_t)row.h * A.osh + (int64_t)row.s * A.oss;
  bool finite = true;
  if (lane < LPR && 4 * lane < A.d_real) {
    f32x4 z = {0.f, 0.f, 0.f, 0.f};
    for (int q = 0; q < GR; ++q) z += *(const f32x4*)(ob[q] + 4 * lane);
    finite = __builtin_isfinite((z[0] + z[1]) + (z[2] + z[3]));
    store_out4<D, E>(A, orow, 4 * lane, z[0] * inv, z[1] * inv, z[2] * inv, z[3] * inv);
  }
  if (A.lse && lane == 0)
    A.lse[(int64_t)b * A.lsb + (int64_t)row.h * A.lsh + row.s] =
        valid ? decode_lse(mt, lt, p < f) : __builtin_nanf("");
  if (valid && wave_any(!finite || !__builtin_isfinite(lt))) {
    __builtin_amdgcn_s_waitcnt(0);
    fix_row<E>(A, b, row.h, kvh, row.s, p, f, sink_end, lane);
  }
}

// The same for the forward's blocks, many rows of few ranges: D / 4 lanes a row
// go through its ranges in turn (65536 rows of two ranges at head_dim 128: 26 us,
// with a workgroup a row 185).
template <int D, Elem E>
__global__ __launch_bounds__(256) void sink_rows_join_kernel(SinkArgs A) {
  constexpr int LPR = D / 4, RPW = 64 / LPR;  // rows a wave
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n_rows = A.groups * A.q_len, n = A.B * A.Hkv * n_rows;
  const int id0 = (blockIdx.x * 4 + wave) * RPW;
  const bool in = id0 + lane / LPR < n;
  const int id = min(id0 + lane / LPR, n - 1);
  const int bkv = id / n_rows, ir = id - bkv * n_rows;
  const int b = bkv / A.Hkv, kvh = bkv - b * A.Hkv;
  const DecodeRow row = decode_row(A, kvh, ir);
  const SeqInfo si = seq_info(A, b);
  const int p = si.base + row.s, dim = 4 * (lane % LPR);
  const int64_t u0 = (((int64_t)bkv * A.row_tiles + (ir >> 4)) * A.splits) * 16 + (ir & 15);
  float mt = -INFINITY;
  for (int s = 0; s < A.splits; ++s) mt = fmaxf(mt, A.part_ml[(u0 + 16 * s) * 3]);
  const float mu = mt == -INFINITY ? 0.f : mt;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  float lt = 0.f, nt = 0.f;
#pragma unroll 4
  for (int s = 0; s < A.splits; ++s) {
    const float* ml = A.part_ml + (u0 + 16 * s) * 3;
    const float w = ml[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[0] - mu);
    if (w != 0.f || ml[1] != ml[1]) {
      lt += w * ml[1];
      nt += w * ml[2];
    }
    y += w * *(const f32x4*)(A.partial + (u0 + 16 * s) * D + dim);
  }
  const bool valid = in && row_valid(A, si, b, row.s);
  const float inv = !valid ? __builtin_nanf("") : p < si.first ? 0.f : 1.f / nt;
  const int64_t orow = (int64_t)b * A.osb + (int64_t)row.h * A.osh + (int64_t)row.s * A.oss;
  bool finite = __builtin_isfinite(lt);
  if (dim < A.d_real) {
    finite &= __builtin_isfinite((y[0] + y[1]) + (y[2] + y[3]));
    if (in) store_out4<D, E>(A, orow, dim, y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
  }
  if (in && A.lse && dim == 0)
    A.lse[(int64_t)b * A.lsb + (int64_t)row.h * A.lsh + row.s] =
        valid ? decode_lse(mt, lt, p < si.first) : __builtin_nanf("");
  // rows that met a non-finite value, again from their own keys
  const uint64_t bad = __builtin_amdgcn_ballot_w64(valid && !finite);
  if (bad) __builtin_amdgcn_s_waitcnt(0);
#pragma unroll 1
  for (int q = 0; q < RPW; ++q) {
    if ((bad >> (LPR * q) & ((uint64_t(1) << LPR) - 1)) == 0) continue;
    const int fid = id0 + q, fkv = fid / n_rows, fb = fkv / A.Hkv, fh = fkv - fb * A.Hkv;
    const DecodeRow fr = decode_row(A, fh, fid - fkv * n_rows);
    const SeqInfo fi = seq_info(A, fb);
    fix_row<E>(A, fb, fr.h, fh, fr.s, fi.base + fr.s, fi.first,
               min(fi.first + A.sinks, A.kv_len), lane);
  }
}

template <int D, Elem E>
hipError_t launch_decode(const SinkArgs& a, hipStream_t stream) {
  const int64_t grid = (int64_t)a.B * a.Hkv * a.row_tiles * a.splits;
  sink_decode_kernel<D, E><<<(unsigned)grid, 256, 0, stream>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  sink_ranges_join_kernel<D, E>
      <<<(unsigned)((int64_t)a.B * a.H * a.q_len), 512, 0, stream>>>(a);
  return hipGetLastError();
}

template <Elem E>
hipError_t launch_elem(const SinkArgs& a, hipStream_t stream) {
  return a.d_real <= 64 ? launch_decode<64, E>(a, stream) : launch_decode<128, E>(a, stream);
}

template <int D, Elem E>
hipError_t launch_rows_join(const SinkArgs& a, hipStream_t stream) {
  constexpr int ROWS = 256 / (D / 4);
  const int64_t rows = (int64_t)a.B * a.H * a.q_len;
  sink_rows_join_kernel<D, E><<<(unsigned)((rows + ROWS - 1) / ROWS), 256, 0, stream>>>(a);
  return hipGetLastError();
}

template <Elem E>
hipError_t rows_join_elem(const SinkArgs& a, hipStream_t stream) {
  return a.d_real <= 64 ? launch_rows_join<64, E>(a, stream) : launch_rows_join<128, E>(a, stream);
}

}  // namespace

hipError_t launch_sink_rows_join(const SinkArgs& a, hipStream_t stream) {
  if (a.elem == (int)Elem::f32) return rows_join_elem<Elem::f32>(a, stream);
  if (a.elem == (int)Elem::bf16) return rows_join_elem<Elem::bf16>(a, stream);
  return rows_join_elem<Elem::f16>(a, stream);
}

hipError_t launch_sink_decode(const SinkArgs& a, hipStream_t stream) {
  (void)hipGetLastError();
  if (a.elem == (int)Elem::f32) return launch_elem<Elem::f32>(a, stream);
  if (a.elem == (int)Elem::bf16) return launch_elem<Elem::bf16>(a, stream);
  return launch_elem<Elem::f16>(a, stream);
}

}  // namespace esa
