// Backward of attention over a causal window with sinks (gfx950), without
// atomics: every gradient is summed in a fixed order.
//
//   P = exp(scale s - lse),  dV = P^T dO,  dP = dO V^T,
//   dS = P * (dP - delta),  delta = rowsum(dO * O),
//   dQ = scale dS K,  dK = scale dS^T Q
//
//   sink_dq_kernel    128 rows a workgroup, over the keys they see, as the
//                     forward: S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T.
//                     First their delta (from O as it was before its rounding,
//                     where the forward kept the difference: a rounded O alone
//                     leaves dQ and dK about 8% further off) and lse in log2
//                     units, left for the next kernel (a kernel of its own for
//                     them read dO once more: 37 us, here 28 more, for 8192
//                     rows of 32 heads of 128)
//   sink_dkdv_kernel  128 keys a workgroup, over the rows that see them: the
//                     lane's own key row (K, V) in registers (or V in LDS), rows
//                     of Q and dO staged in LDS: S = Q K^T, dP = dO V^T, dV^T += dO^T P,
//                     dK^T += Q^T dS
//   sink_join_kernel  blocks whose rows were split: the parts in order
//
// Key blocks start at the sequence's first key, so the sinks are in the first
// ones.  A block's rows are those of every query head of the kv group, one
// after the other, and may be cut into chunks, one workgroup each, that leave
// float32 parts: a sink's block, which every later row sees, and the blocks
// that would run as an unfilled last round of the grid (sink_bwd_plan).
//
// Bound: registers, and with them waves: dK, dV and K of 32 keys take 160 of a
// wave's 256 at head_dim 128, so two waves a SIMD share its pipes and wait for
// each other's products (of dK / dV's cycles the matrix pipe works 50%, of
// dQ's 42%).  V in LDS leaves dK / dV room to read each operand three products
// ahead and to place the exponentials and dS beside products: with V in
// registers and one product after the other 365 us, so 275 (8192 rows, 32 heads
// on 8, window 1024, bf16: 930 TFLOP/s of its four products); dQ, a pipeline of
// 32-key stages as the forward, 240 against 262 with 64-key stages and no
// pipeline (700 TFLOP/s of its three), 20 of it the rows' delta.  8 padded
// sequences of 4099, 16 heads of 64, window 500, f16: 194 and 167; float32, 2 x
// 2048 rows, 8 heads of 64, window 256: 76 (and 100 against 114 with one wave a
// SIMD, before its grid was cut for 256 slots) and 54.
#include <algorithm>

#include "esa_sink.hpp"

namespace esa {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

template <int D, Elem E>
struct SinkBwdCfg {
  // waves a SIMD: what the registers allow (dK / dV at head_dim 64 in 16 bits
  // gains nothing from a third: 195 us against 191)
  static constexpr int DQ_WAVES = E == Elem::f32 ? (D >= 128 ? 1 : 2) : D >= 128 ? 2 : 3;
  static constexpr int KV_WAVES = E == Elem::f32 && D >= 128 ? 1 : 2;
  // dK / dV: where K, V, their gradients and the products take more registers
  // than half a SIMD's, V's rows are kept in LDS, and stages are 32 rows, so that
  // two workgroups' still fit
  static constexpr bool V_LDS = KV_WAVES == 2 && (E == Elem::f32 || D >= 128);
  static constexpr int ROWS = E == Elem::f32 || D >= 128 ? 32 : 64;
};

template <Elem E>
__device__ __forceinline__ const typename ElemT<E>::T* at(const void* p, int64_t off) {
  return (const typename ElemT<E>::T*)p + off;
}

// dQ of one row from its own keys, by one wave
template <Elem E>
__device__ void fix_dq_row(const SinkArgs& A, int b, int h, int kvh, int row, int p, int f,
                           int sink_end, int lane) {
  using T = ElemT<E>;
  const auto* q = at<E>(A.q, (int64_t)b * A.qsb + (int64_t)h * A.qsh + (int64_t)row * A.qss);
  const auto* g = at<E>(A.dout, (int64_t)b * A.dosb + (int64_t)h * A.dosh + (int64_t)row * A.doss);
  const auto* k = at<E>(A.k, (int64_t)b * A.ksb + (int64_t)kvh * A.ksh);
  const auto* v = at<E>(A.v, (int64_t)b * A.vsb + (int64_t)kvh * A.vsh);
  const int64_t st = ((int64_t)b * A.H + h) * A.qpad + row;
  const float lse2 = A.lse2[st], delta = A.delta[st];
  const RowKeys rk = row_keys(p, f, A.window, sink_end);
  float acc[2] = {0.f, 0.f};
#pragma unroll 1
  for (int i0 = 0; i0 < rk.n; i0 += 64) {
    float ds = 0.f;
    if (i0 + lane < rk.n) {
      const int64_t j = rk.key(i0 + lane);
      const float s = row_dot<E>(q, k + j * A.kss, A.d_real) * A.scale_log2;
      const float dp = row_dot<E>(g, v + j * A.vss, A.d_real);
      ds = __builtin_amdgcn_exp2f(s - lse2) * (dp - delta) * A.sm_scale;
    }
    const int n = min(64, rk.n - i0);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const float w = __shfl(ds, i, 64);
      const auto* kr = k + (int64_t)rk.key(i0 + i) * A.kss;
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (lane + 64 * c < A.d_real)
          acc[c] = __builtin_fmaf(w, T::load(kr + lane + 64 * c), acc[c]);
    }
  }
  auto* dq = (typename T::T*)A.dq + (int64_t)b * A.dqsb + (int64_t)h * A.dqsh + (int64_t)row * A.dqss;
#pragma unroll
  for (int c = 0; c < 2; ++c)
    if (lane + 64 * c < A.d_real) T::store(dq + lane + 64 * c, acc[c]);
}

template <int D, int DR, Elem E>
__global__ __launch_bounds__(256, (SinkBwdCfg<D, E>::DQ_WAVES)) void sink_dq_kernel(
    SinkArgs A) {
  using T = SinkTile<D, E, false, DR>;
  using Stage = SinkStage<D, E, 32, 256>;
  using LdsT = typename T::LdsT;
  constexpr int ND = T::ND, N = 32 * D;
  // four stages of 32 keys, as the forward's
  __shared__ __attribute__((aligned(1024))) LdsT k0_[N];
  __shared__ __attribute__((aligned(1024))) LdsT v0_[N];
  __shared__ __attribute__((aligned(1024))) LdsT k1_[N];
  __shared__ __attribute__((aligned(1024))) LdsT v1_[N];
  __shared__ __attribute__((aligned(1024))) LdsT k2_[N];
  __shared__ __attribute__((aligned(1024))) LdsT v2_[N];
  __shared__ __attribute__((aligned(1024))) LdsT k3_[N];
  __shared__ __attribute__((aligned(1024))) LdsT v3_[N];

  const RowItem it = row_item(A);
  const int b = it.b, h = it.h, kvh = it.kvh, r0 = it.qb * 128;
  const SeqInfo si = seq_info(A, b);
  const int f = si.first, sink_end = min(f + A.sinks, A.kv_len), W = A.window;
  const KeyStages keys = key_stages(A, si, r0, sink_end);

  const int tid = threadIdx.x;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hf = lane >> 5;
  const int r = r0 + wave * 32 + l32;
  const bool row_in = r < A.q_len;
  const int p = si.base + r;
  const int pb = keys.pb, pw0 = si.base + r0 + wave * 32, pw1 = min(pw0 + 31, pb);
  const int n_all = keys.n_all;
  const WaveStages ws = wave_stages(keys, pw0, pw1, W, sink_end);

  Stage ks, vs;
  ks.init(at<E>(A.k, (int64_t)b * A.ksb + (int64_t)kvh * A.ksh), A.kss, A.kv_len, A.d_real, tid);
  vs.init(at<E>(A.v, (int64_t)b * A.vsb + (int64_t)kvh * A.vsh), A.vss, A.kv_len, A.d_real, tid);
  auto issue = [&](int i, LdsT* kd, LdsT* vd) __attribute__((always_inline)) {
    if (i < n_all) {
      ks.issue(keys.key0(i), kd, wave);
      vs.issue(keys.key0(i), vd, wave);
    }
  };

  T t;
  t.init(lane);
  typename T::Frag qf, gf;
  t.load_frag(qf, at<E>(A.q, (int64_t)b * A.qsb + (int64_t)h * A.qsh + (int64_t)r * A.qss), row_in,
              A.d_real);
  t.load_frag(gf, at<E>(A.dout, (int64_t)b * A.dosb + (int64_t)h * A.dosh + (int64_t)r * A.doss),
              row_in, A.d_real);
  float lse2 = 0.f, delta = 0.f;
  {
    const int64_t at_o = (int64_t)b * A.osb + (int64_t)h * A.osh + (int64_t)r * A.oss;
    typename T::Frag o, res;
    t.load_frag(o, at<E>(A.o, at_o), row_in, A.d_real);
    t.load_frag(res, at<E>(A.ores, at_o), row_in && A.ores, A.d_real);
    const float lse = row_in ? A.lse[(int64_t)b * A.lsb + (int64_t)h * A.lsh + r] : 0.f;
    delta = T::dot(o, gf, T::dot(res, gf, 0.f));
    delta += __shfl_xor(delta, 32, 64);
    // a row that sees nothing: kept finite, so its masked scores give P = 0
    lse2 = lse == -INFINITY ? -3.0e38f : lse * kLog2e;
    if (row_in && hf == 0) {
      const int64_t st = ((int64_t)b * A.H + h) * A.qpad + r;
      A.delta[st] = delta;
      A.lse2[st] = lse2;
    }
  }
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
  const float scale = A.scale_log2;

  // A pipeline over the stages: s holds the coming stage's scores (of the keys
  // that the wave sees); its exponentials run beside the product dP, dS beside
  // the next stage's scores, dQ's product last.
  f32x16 s = f32x16{};
  bool used = false;
  auto hide = [&](f32x16& x, int i) __attribute__((always_inline)) {
    if (!ws.full(i)) {
      uint32_t m[16];
      key_masks<0>(m, seen_keys(p, keys.key0(i), W, sink_end) >> (4 * hf));
      mask_select(x, m);
    }
  };
  // stage i: its K and V, the next stage's K
  auto step = [&](const LdsT* kbuf, const LdsT* vbuf, const LdsT* knext, int i)
                  __attribute__((always_inline)) {
    const bool next = ws.sees(i + 1);
    if (!used) {
      if (next) {
        s = f32x16{};
        t.row_product(s, knext, 0, qf);
        hide(s, i + 1);
      }
      used = next;
      return;
    }
    f32x16 sn = f32x16{}, dp = f32x16{};
    if constexpr (T::ES == 2) {
      // in written order, operands read AHEAD products ahead
      constexpr int AHEAD = 4, NS = T::NS;
      typename T::V8 va[NS], ka[NS];
      u32x4 kc[NS];
      typename T::P pd;
      auto read = [&](int i) __attribute__((always_inline)) {
        const int k = i % NS;
        if (i < NS)
          va[k] = t.row_operand(vbuf, 0, k);
        else if (i < 2 * NS)
          ka[k] = t.row_operand(knext, 0, k);
        else if (i < 3 * NS)
          kc[k] = t.col_operand(kbuf, 0, k % ND, k / ND);
      };
      auto grads = [&](int k) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 8 * k / NS; q < 8 * (k + 1) / NS; ++q) {  // pairs of keys (rows)
#pragma unroll
          for (int e = 2 * q; e < 2 * q + 2; ++e) s[e] *= dp[e] - delta;
          pd.w[q] = T::M::pack2(s[2 * q], s[2 * q + 1]);
        }
      };
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) read(k);
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        dp = T::M::mfma32(va[k], gf.f[k], dp);
        read(k + AHEAD);
#pragma unroll
        for (int e = 2 * (8 * k / NS); e < 2 * (8 * (k + 1) / NS); ++e)
          s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], scale, -lse2));
      }
      // (past the wave's last key: of whatever the buffer holds, and dropped)
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        sn = T::M::mfma32(ka[k], qf.f[k], sn);
        read(NS + k + AHEAD);
        if (k > 0) grads(k - 1);
      }
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        if (k == 0) grads(NS - 1);
        T::col_step(acc[k % ND], kc[k], pd, k / ND);
        read(2 * NS + k + AHEAD);
      }
      __builtin_amdgcn_sched_barrier(0);
    } else {
      t.row_product(dp, vbuf, 0, gf);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], scale, -lse2)) * (dp[e] - delta);
      t.row_product(sn, knext, 0, qf);
      t.col_product(acc, kbuf, 0, t.pack(s));
    }
    if (next) hide(sn, i + 1);
    s = sn;
    used = next;
  };
  auto ready = [&](int i) __attribute__((always_inline)) {
    if (i + 2 < n_all)
      stage_wait<2 * Stage::LOADS>();
    else
      stage_wait<0>();
  };
  issue(0, k0_, v0_);
  issue(1, k1_, v1_);
  issue(2, k2_, v2_);
  if (n_all > 0) {
    if (n_all > 2)
      stage_wait<4 * Stage::LOADS>();
    else
      stage_wait<0>();
    if (ws.sees(0)) {
      t.row_product(s, k0_, 0, qf);
      hide(s, 0);
      used = true;
    }
  }
  for (int i = 0; i < n_all; i += 4) {
    ready(i);
    issue(i + 3, k3_, v3_);
    step(k0_, v0_, k1_, i);
    if (i + 1 >= n_all) break;
    ready(i + 1);
    issue(i + 4, k0_, v0_);
    step(k1_, v1_, k2_, i + 1);
    if (i + 2 >= n_all) break;
    ready(i + 2);
    issue(i + 5, k1_, v1_);
    step(k2_, v2_, k3_, i + 2);
    if (i + 3 >= n_all) break;
    ready(i + 3);
    issue(i + 6, k2_, v2_);
    step(k3_, v3_, k0_, i + 3);
  }

  const bool met = row_in && !sum_finite(acc);
  auto* dq = (typename ElemT<E>::T*)A.dq + (int64_t)b * A.dqsb + (int64_t)h * A.dqsh +
             (int64_t)r * A.dqss;
#pragma unroll
  for (int d = 0; d < ND; ++d)
    T::store32(dq, 32 * d, acc[d], A.sm_scale, hf, A.d_real, row_in);
  uint64_t bad = __builtin_amdgcn_ballot_w64(met);
  bad = (bad | bad >> 32) & 0xffffffffull;
  if (bad) __builtin_amdgcn_s_waitcnt(0);  // the stores above come first
  while (bad) {
    const int i = __builtin_ctzll(bad);
    bad &= bad - 1;
    const int row = r0 + wave * 32 + i;
    fix_dq_row<E>(A, b, h, kvh, row, min(si.base + row, A.kv_len - 1), f, sink_end, lane);
  }
}

// One key block's work: which rows, how they are cut.
struct KeyItem {
  int b, kvh, kblk, chunk, n_chunks;
  int64_t part;  // index of its float32 part
};
// parts a kv head keeps
__device__ __host__ __forceinline__ int kv_parts(const SinkArgs& A) {
  int n = 0;
  for (int c = 0; c < 3; ++c) n += A.cls_cut[c] > 1 ? A.cls_n[c] * A.cls_cut[c] : 0;
  return n;
}
// Block `block` of class `cls` of kv head bkv (over the batch), one chunk of it
__device__ __forceinline__ KeyItem key_block(const SinkArgs& A, int bkv, int cls, int block,
                                             int chunk) {
  KeyItem k;
  k.b = bkv / A.Hkv;
  k.kvh = bkv - k.b * A.Hkv;
  k.kblk = block;
  k.chunk = chunk;
  k.n_chunks = A.cls_cut[cls];
  int at = block * k.n_chunks + chunk;
  for (int c = 0; c < cls; ++c) {
    k.kblk += A.cls_n[c];
    at += A.cls_cut[c] > 1 ? A.cls_n[c] * A.cls_cut[c] : 0;
  }
  k.part = (int64_t)bkv * kv_parts(A) + at;
  return k;
}
// The grid's order: class by class (the longest work first), the kv heads of
// an XCD's run (or all of them) in each class one after the other.
__device__ __forceinline__ KeyItem key_item(const SinkArgs& A) {
  int item = blockIdx.x, n_kv = A.B * A.Hkv, kv0 = 0;
  if (A.xcd_runs) {
    n_kv >>= 3;
    kv0 = (item & 7) * n_kv;
    item >>= 3;
  }
  int cls = 0;
  for (; cls < 2; ++cls) {
    const int n = n_kv * A.cls_n[cls] * A.cls_cut[cls];
    if (item < n) break;
    item -= n;
  }
  const int per = A.cls_n[cls] * A.cls_cut[cls];
  const int kv = item / per, u = item - kv * per;
  const int block = u / A.cls_cut[cls];
  return key_block(A, kv0 + kv, cls, block, u - block * A.cls_cut[cls]);
}

// Stores 32 keys' dK^T and dV^T (one wave's accumulators; in: the lane's key is one)
template <int D, int DR, Elem E>
__device__ __forceinline__ void store_keys(const SinkArgs& A, int b, int kvh, int j, int hf,
                                           const f32x16 (&dk)[DR / 32],
                                           const f32x16 (&dv)[DR / 32], bool in) {
  using T = SinkTile<D, E>;
  auto* kr = (typename ElemT<E>::T*)A.dk + (int64_t)b * A.dksb + (int64_t)kvh * A.dksh +
             (int64_t)j * A.dkss;
  auto* vr = (typename ElemT<E>::T*)A.dv + (int64_t)b * A.dvsb + (int64_t)kvh * A.dvsh +
             (int64_t)j * A.dvss;
#pragma unroll
  for (int d = 0; d < DR / 32; ++d) {
    T::store32(kr, 32 * d, dk[d], A.sm_scale, hf, A.d_real, in);
    T::store32(vr, 32 * d, dv[d], 1.f, hf, A.d_real, in);
  }
}

// dK and dV of one key from the rows that see it, by one wave
template <Elem E>
__device__ void fix_key(const SinkArgs& A, const SeqInfo& si, int b, int kvh, int j, int sink_end,
                        int lane) {
  using T = ElemT<E>;
  const auto* k = at<E>(A.k, (int64_t)b * A.ksb + (int64_t)kvh * A.ksh + (int64_t)j * A.kss);
  const auto* v = at<E>(A.v, (int64_t)b * A.vsb + (int64_t)kvh * A.vsh + (int64_t)j * A.vss);
  const int p_last = min(si.base + A.q_len, A.kv_len) - 1;
  const int hi = j < sink_end ? p_last : min(p_last, j + A.window - 1);
  const int lo = max(j, si.base);
  float ak[2] = {0.f, 0.f}, av[2] = {0.f, 0.f};
#pragma unroll 1
  for (int h = kvh * A.groups; h < (kvh + 1) * A.groups; ++h) {
    const auto* q = at<E>(A.q, (int64_t)b * A.qsb + (int64_t)h * A.qsh);
    const auto* g = at<E>(A.dout, (int64_t)b * A.dosb + (int64_t)h * A.dosh);
    const int64_t st = ((int64_t)b * A.H + h) * A.qpad;
#pragma unroll 1
    for (int p0 = lo; p0 <= hi; p0 += 64) {
      float pr = 0.f, ds = 0.f;
      if (p0 + lane <= hi) {
        const int64_t r = p0 + lane - si.base;
        const float s = row_dot<E>(q + r * A.qss, k, A.d_real) * A.scale_log2;
        const float dp = row_dot<E>(g + r * A.doss, v, A.d_real);
        pr = __builtin_amdgcn_exp2f(s - A.lse2[st + r]);
        ds = pr * (dp - A.delta[st + r]) * A.sm_scale;
      }
      const int n = min(64, hi - p0 + 1);
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const float wp = __shfl(pr, i, 64), wd = __shfl(ds, i, 64);
        const int64_t r = p0 + i - si.base;
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (lane + 64 * c < A.d_real) {
            ak[c] = __builtin_fmaf(wd, T::load(q + r * A.qss + lane + 64 * c), ak[c]);
            av[c] = __builtin_fmaf(wp, T::load(g + r * A.doss + lane + 64 * c), av[c]);
          }
      }
    }
  }
  auto* kr = (typename T::T*)A.dk + (int64_t)b * A.dksb + (int64_t)kvh * A.dksh + (int64_t)j * A.dkss;
  auto* vr = (typename T::T*)A.dv + (int64_t)b * A.dvsb + (int64_t)kvh * A.dvsh + (int64_t)j * A.dvss;
#pragma unroll
  for (int c = 0; c < 2; ++c)
    if (lane + 64 * c < A.d_real) {
      T::store(kr + lane + 64 * c, ak[c]);
      T::store(vr + lane + 64 * c, av[c]);
    }
}

// The keys of a wave whose sums came out non-finite, again (j0: its first key)
template <Elem E>
__device__ __forceinline__ void fix_keys(const SinkArgs& A, const SeqInfo& si, int b, int kvh,
                                         int j0, int sink_end, bool met, int lane) {
  uint64_t bad = __builtin_amdgcn_ballot_w64(met);
  bad = (bad | bad >> 32) & 0xffffffffull;
  if (bad) __builtin_amdgcn_s_waitcnt(0);  // the stores above come first
  while (bad) {
    const int i = __builtin_ctzll(bad);
    bad &= bad - 1;
    fix_key<E>(A, si, b, kvh, j0 + i, sink_end, lane);
  }
}

template <int D, int DR, Elem E>
__global__ __launch_bounds__(256, (SinkBwdCfg<D, E>::KV_WAVES)) void sink_dkdv_kernel(
    SinkArgs A) {
  using C = SinkBwdCfg<D, E>;
  using T = SinkTile<D, E, (D >= 128), DR>;
  using Stage = SinkStage<D, E, C::ROWS, 256>;
  using LdsT = typename T::LdsT;
  constexpr int ND = T::ND;
  __shared__ __attribute__((aligned(1024))) LdsT q_st0[C::ROWS * D];
  __shared__ __attribute__((aligned(1024))) LdsT g_st0[C::ROWS * D];
  __shared__ __attribute__((aligned(1024))) LdsT q_st1[C::ROWS * D];
  __shared__ __attribute__((aligned(1024))) LdsT g_st1[C::ROWS * D];
  __shared__ __attribute__((aligned(16))) typename T::Frag v_rows[C::V_LDS ? 256 : 1];
  __shared__ __attribute__((aligned(256))) float stat0[2 * 64];  // lse2, then delta
  __shared__ __attribute__((aligned(256))) float stat1[2 * 64];

  const KeyItem it = key_item(A);
  const int b = it.b, kvh = it.kvh;
  const SeqInfo si = seq_info(A, b);
  const int f = si.first, sink_end = min(f + A.sinks, A.kv_len), W = A.window;

  const int tid = threadIdx.x;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hf = lane >> 5;

  // keys before the sequence's first one: no row sees them
  if (it.chunk == 0) {
    const int z1 = min(f, min(it.kblk * 128 + 128, A.kv_len));
    for (int j = it.kblk * 128 + (tid >> 4); j < z1; j += 16) {
      auto* kr = (typename ElemT<E>::T*)A.dk + (int64_t)b * A.dksb + (int64_t)kvh * A.dksh +
                 (int64_t)j * A.dkss;
      auto* vr = (typename ElemT<E>::T*)A.dv + (int64_t)b * A.dvsb + (int64_t)kvh * A.dvsh +
                 (int64_t)j * A.dvss;
      for (int d = 4 * (tid & 15); d < A.d_real; d += 64) {
        T::store4(kr, d, 0.f, 0.f, 0.f, 0.f);
        T::store4(vr, d, 0.f, 0.f, 0.f, 0.f);
      }
    }
  }
  const int j0 = f + it.kblk * 128;
  if (j0 >= A.kv_len) return;

  // ---- the rows that see the block, as stages of every query head in turn;
  // this workgroup's share of them
  const int p_last = min(si.base + A.q_len, A.kv_len) - 1;
  const int p_lo = max(j0, si.base);
  const int p_hi = j0 < sink_end ? p_last : min(p_last, j0 + 127 + W - 1);
  const int per_head = p_hi >= p_lo ? (p_hi - p_lo) / C::ROWS + 1 : 0;
  const int64_t total = (int64_t)per_head * A.groups;
  const int s0 = (int)(total * it.chunk / it.n_chunks);
  const int s1 = (int)(total * (it.chunk + 1) / it.n_chunks);

  const int jw0 = j0 + wave * 32;  // the wave's first key
  const int j = jw0 + l32;
  const bool key_in = j < A.kv_len;

  T t;
  t.init(lane);
  typename T::Frag kf, vf;
  t.load_frag(kf, at<E>(A.k, (int64_t)b * A.ksb + (int64_t)kvh * A.ksh + (int64_t)j * A.kss),
              key_in, A.d_real);
  t.load_frag(vf, at<E>(A.v, (int64_t)b * A.vsb + (int64_t)kvh * A.vsh + (int64_t)j * A.vss),
              key_in, A.d_real);
  // (a lane reads back what it wrote)
  constexpr int PIECES = sizeof(vf) / 16;
  u32x4* const v_own = (u32x4*)v_rows + (wave * PIECES * 64 + lane);
  if constexpr (C::V_LDS) {
#pragma unroll
    for (int s = 0; s < PIECES; ++s) v_own[64 * s] = __builtin_bit_cast(u32x4, vf.f[s]);
  }
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dk[d] = dv[d] = f32x16{};
  const float scale = A.scale_log2;

  Stage qs, gs;
  qs.init(nullptr, A.qss, A.q_len, A.d_real, tid);
  gs.init(nullptr, A.doss, A.q_len, A.d_real, tid);
  int head = per_head > 0 ? s0 / per_head : 0, at_stage = s0 - head * per_head;
  int staged = -1;
  // Stage `at` of a head is, of the block's, the one whose number among all rows
  // is at modulo per_head: blocks that run side by side read the same rows at the
  // same time (8192 rows of 4 heads, window 1024: 875 MB from beyond L2, 350 so)
  const int turn = per_head > 0 ? (p_lo - si.base) / C::ROWS % per_head : 0;
  // the next stage in order -> buffers; returns its first row
  auto issue = [&](LdsT* qd, LdsT* gd, float* stat) __attribute__((always_inline)) {
    const int h = kvh * A.groups + head;
    const int k = at_stage - turn + (at_stage < turn ? per_head : 0);
    const int row0 = p_lo - si.base + k * C::ROWS;
    if (h != staged) {  // another head's rows
      qs.rebase(at<E>(A.q, (int64_t)b * A.qsb + (int64_t)h * A.qsh));
      gs.rebase(at<E>(A.dout, (int64_t)b * A.dosb + (int64_t)h * A.dosh));
      staged = h;
    }
    qs.issue(row0, qd, wave);
    gs.issue(row0, gd, wave);
    // lse2 and delta, 64 rows each, zeros past q_len: copied to LDS like the
    // rows, so the whole issue runs without a divergent branch (a branch here
    // had the compiler save a value for all lanes under the branch's mask)
    if (wave < 2) {
      const float* src = (wave ? A.delta : A.lse2) + ((int64_t)b * A.H + h) * A.qpad;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          (void*)src, (short)0, A.q_len * 4, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(stat + wave * 64), 4, lane * 4,
                                               row0 * 4, 0, 0);
    }
    if (++at_stage == per_head) {
      at_stage = 0;
      ++head;
    }
    return row0;
  };
  auto block = [&](const LdsT* qb, const LdsT* gb, const float* stat, int rb, int row0)
                   __attribute__((always_inline)) {
    const int p0 = si.base + row0 + 32 * rb, p1 = min(p0 + 31, p_last);
    if (p0 > p_last || none_seen(p0, p1, jw0, W, sink_end)) return;
    const bool whole = p0 + 31 <= p_last && all_seen(p0, p0 + 31, jw0, W, sink_end);
    auto hide = [&](f32x16& s) __attribute__((always_inline)) {
      uint32_t m[16];
      key_masks<0>(m, seen_rows(j, p0, p_last, W, sink_end) >> (4 * hf));
      mask_select(s, m);
    };
    auto row_stat = [&](int at, int q4) __attribute__((always_inline)) {
      return *(const f32x4*)(stat + at + 32 * rb + 8 * q4 + 4 * hf);
    };
    f32x16 s = f32x16{}, dp = f32x16{};
    if constexpr (T::ES == 2) {
      // The four products in written order, each beside the vector work of the
      // one before it (S: none; dP: P's exponentials; dV: dS; dK: dS's rest),
      // operands read AHEAD products ahead.
      constexpr int AHEAD = 3, NS = T::NS;  // products of each
      typename T::V8 qa[NS], ga[NS], va[NS];
      int base;  // of the reads' addresses
      u32x4 gc[NS], qc[NS];
      typename T::P pp, pd;
      f32x4 l2[4], dl[4];
      // beside product k: the lse or delta of the four rows after its own pairs'
      auto ahead_stat = [&](f32x4 (&to)[4], int at, int k) __attribute__((always_inline)) {
#pragma unroll
        for (int q4 = 1; q4 < 4; ++q4)
          if (2 * q4 - 2 >= 8 * k / NS && 2 * q4 - 2 < 8 * (k + 1) / NS) to[q4] = row_stat(at, q4);
      };
      auto read = [&](int i) __attribute__((always_inline)) {  // operands in their order
        const int k = i % NS;
        if (i < 2 * NS) {
          if (k == 0) base = T::fresh(t.ra[0]);
          if (i < NS) {
            qa[k] = t.row_operand(qb, rb, k, base);
          } else {
            ga[k] = t.row_operand(gb, rb, k, base);
            if constexpr (C::V_LDS) va[k] = __builtin_bit_cast(typename T::V8, v_own[64 * k]);
          }
        } else if (i < 4 * NS) {
          if (k % ND == 0) base = T::fresh(t.ca[0]);
          if (i < 3 * NS)
            gc[k] = t.col_operand(gb, rb, k % ND, k / ND, base);
          else
            qc[k] = t.col_operand(qb, rb, k % ND, k / ND, base);
        }
      };
      auto exps = [&](int k) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 8 * k / NS; q < 8 * (k + 1) / NS; ++q) {  // pairs of keys (rows)
#pragma unroll
          for (int e = 2 * q; e < 2 * q + 2; ++e)
            s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], scale, -l2[e / 4][e % 4]));
          pp.w[q] = T::M::pack2(s[2 * q], s[2 * q + 1]);
        }
      };
      auto grads = [&](int k) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 8 * k / NS; q < 8 * (k + 1) / NS; ++q) {  // pairs of keys (rows)
#pragma unroll
          for (int e = 2 * q; e < 2 * q + 2; ++e) s[e] *= dp[e] - dl[e / 4][e % 4];
          pd.w[q] = T::M::pack2(s[2 * q], s[2 * q + 1]);
        }
      };
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) read(k);
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        s = T::M::mfma32(qa[k], kf.f[k], s);
        read(k + AHEAD);
      }
      l2[0] = row_stat(0, 0);
      __builtin_amdgcn_sched_barrier(0);
      if (!whole) hide(s);
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        dp = T::M::mfma32(ga[k], C::V_LDS ? va[k] : vf.f[k], dp);
        read(NS + k + AHEAD);
        ahead_stat(l2, 0, k);
        if (k > 0) exps(k - 1);
      }
      dl[0] = row_stat(64, 0);
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        T::col_step(dv[k % ND], gc[k], pp, k / ND);
        read(2 * NS + k + AHEAD);
        ahead_stat(dl, 64, k);
        if (k == 0) exps(NS - 1);
        if (k > 0) grads(k - 1);
      }
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        if (k == 0) grads(NS - 1);
        T::col_step(dk[k % ND], qc[k], pd, k / ND);
        read(3 * NS + k + AHEAD);
      }
      __builtin_amdgcn_sched_barrier(0);
    } else {
      t.row_product(s, qb, rb, kf);
      __builtin_amdgcn_sched_barrier(0);
      if (!whole) hide(s);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 l2 = row_stat(0, q);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s[4 * q + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * q + e], scale, -l2[e]));
      }
      if constexpr (C::V_LDS) {
#pragma unroll
        for (int s = 0; s < PIECES; ++s) vf.f[s] = __builtin_bit_cast(f32x4, v_own[64 * s]);
      }
      t.row_product(dp, gb, rb, vf);
      __builtin_amdgcn_sched_barrier(0);
      t.col_product(dv, gb, rb, t.pack(s));
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 dl = row_stat(64, q);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * q + e] = s[4 * q + e] * (dp[4 * q + e] - dl[e]);
      }
      t.col_product(dk, qb, rb, t.pack(dp));
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  int row_a = 0, row_b = 0;
  if (s0 < s1) row_a = issue(q_st0, g_st0, stat0);
  for (int i = s0; i < s1; i += 2) {
    stage_ready();
    if (i + 1 < s1) row_b = issue(q_st1, g_st1, stat1);
#pragma unroll
    for (int rb = 0; rb < C::ROWS / 32; ++rb) block(q_st0, g_st0, stat0, rb, row_a);
    if (i + 1 >= s1) break;
    stage_ready();
    if (i + 2 < s1) row_a = issue(q_st0, g_st0, stat0);
#pragma unroll
    for (int rb = 0; rb < C::ROWS / 32; ++rb) block(q_st1, g_st1, stat1, rb, row_b);
  }

  if (it.n_chunks > 1) {  // a part: [wave][dK, dV][d block][register][lane]
    float* part = A.partial + (it.part * 4 + wave) * (2 * ND * 16 * 64) + lane;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        part[(d * 16 + e) * 64] = dk[d][e];
        part[((ND + d) * 16 + e) * 64] = dv[d][e];
      }
    return;
  }
  const bool met = key_in && !(sum_finite(dk) && sum_finite(dv));
  store_keys<D, DR, E>(A, b, kvh, j, hf, dk, dv, key_in);
  fix_keys<E>(A, si, b, kvh, jw0, sink_end, met, lane);
}

// The parts of one cut key block's 32 keys, summed in their order: each wave
// takes the 32-dim pieces of dK and dV in turn.
template <int D, int DR, Elem E>
__global__ __launch_bounds__(256) void sink_join_kernel(SinkArgs A) {
  using T = SinkTile<D, E, false, DR>;
  constexpr int ND = T::ND;
  __shared__ uint32_t met[4][32];
  int n_cut = 0;
  for (int c = 0; c < 3; ++c) n_cut += A.cls_cut[c] > 1 ? A.cls_n[c] : 0;
  const int quarter = blockIdx.x & 3, bkv = (blockIdx.x >> 2) / n_cut;
  int block = (blockIdx.x >> 2) - bkv * n_cut, cls = 0;
  for (; cls < 2; ++cls) {
    const int n = A.cls_cut[cls] > 1 ? A.cls_n[cls] : 0;
    if (block < n) break;
    block -= n;
  }
  const KeyItem it = key_block(A, bkv, cls, block, 0);
  const int n = it.n_chunks;
  const SeqInfo si = seq_info(A, it.b);
  const int sink_end = min(si.first + A.sinks, A.kv_len);
  const int tid = threadIdx.x;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hf = lane >> 5;
  const int jw0 = si.first + it.kblk * 128 + quarter * 32;
  if (jw0 >= A.kv_len) return;  // (the whole workgroup)
  const int j = jw0 + l32;
  const bool key_in = j < A.kv_len;
  bool bad = false;
  for (int w = wave; w < 2 * ND; w += 4) {  // dK's pieces, then dV's
    f32x16 x = f32x16{};
    const float* part = A.partial + (it.part * 4 + quarter) * (2 * ND * 16 * 64) +
                        w * (16 * 64) + lane;
    // (four parts on their way at a time, added in order)
    constexpr int64_t STEP = 4 * 2 * ND * 16 * 64;
    int c = 0;
    for (; c + 4 <= n; c += 4, part += 4 * STEP) {
      float y[4][16];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) y[u][e] = part[u * STEP + e * 64];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] += y[u][e];
    }
    for (; c < n; ++c, part += STEP)
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] += part[e * 64];
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) sum += x[e];
    bad |= !__builtin_isfinite(sum);
    const bool is_k = w < ND;
    const int d = is_k ? w : w - ND;
    const float scale = is_k ? A.sm_scale : 1.f;
    auto* row = is_k ? (typename ElemT<E>::T*)A.dk + (int64_t)it.b * A.dksb +
                           (int64_t)it.kvh * A.dksh + (int64_t)j * A.dkss
                     : (typename ElemT<E>::T*)A.dv + (int64_t)it.b * A.dvsb +
                           (int64_t)it.kvh * A.dvsh + (int64_t)j * A.dvss;
    T::store32(row, 32 * d, x, scale, hf, A.d_real, key_in);
  }
  // a key that met a non-finite value, again from its own rows (by one wave,
  // after every wave's stores)
  uint64_t any = __builtin_amdgcn_ballot_w64(bad && key_in);
  any = (any | any >> 32) & 0xffffffffull;
  if (lane < 32) met[wave][lane] = (uint32_t)(any >> lane) & 1u;
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  const bool fix = wave == 0 && (met[0][l32] | met[1][l32] | met[2][l32] | met[3][l32]);
  fix_keys<E>(A, si, it.b, it.kvh, jw0, sink_end, fix, lane);
}

template <int D, int DR, Elem E>
hipError_t launch_bwd(const SinkArgs& a, hipStream_t stream) {
  SinkArgs g = a;
  const int64_t n_dq = (int64_t)a.B * a.H * a.nqb;
  g.xcd_runs = sink_xcd_runs(a, n_dq);
  sink_dq_kernel<D, DR, E><<<(unsigned)n_dq, 256, 0, stream>>>(g);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  int64_t units = 0, n_cut = 0;
  for (int c = 0; c < 3; ++c) {
    units += (int64_t)a.cls_n[c] * a.cls_cut[c];
    n_cut += a.cls_cut[c] > 1 ? a.cls_n[c] : 0;
  }
  const int64_t n_kv = (int64_t)a.B * a.Hkv * units;
  g.xcd_runs = sink_xcd_runs(a, n_kv);
  sink_dkdv_kernel<D, DR, E><<<(unsigned)n_kv, 256, 0, stream>>>(g);
  e = hipGetLastError();
  if (e != hipSuccess || n_cut == 0) return e;
  sink_join_kernel<D, DR, E><<<(unsigned)(4 * a.B * a.Hkv * n_cut), 256, 0, stream>>>(g);
  return hipGetLastError();
}

template <Elem E>
hipError_t launch_elem(const SinkArgs& a, hipStream_t stream) {
  if (a.d_real <= 64) return launch_bwd<64, 64, E>(a, stream);
  return a.d_real <= 96 ? launch_bwd<128, 96, E>(a, stream) : launch_bwd<128, 128, E>(a, stream);
}

}  // namespace

hipError_t launch_sink_bwd(const SinkArgs& a, hipStream_t stream) {
  (void)hipGetLastError();
  if (a.elem == (int)Elem::f32) return launch_elem<Elem::f32>(a, stream);
  if (a.elem == (int)Elem::bf16) return launch_elem<Elem::bf16>(a, stream);
  return launch_elem<Elem::f16>(a, stream);
}

}  // namespace esa
