// Forward of attention over a causal window with sinks (gfx950).
//
//   s = scale q k^T on visible keys,  o = softmax(s) v,  lse = log sum exp(s)
//
// One workgroup (4 waves) takes 128 rows of one (sequence, head) and walks
// the keys they see: the sinks' blocks, then the window's, or one run of
// blocks where the two meet.  Each wave holds 32 rows: Q in registers, O^T in
// accumulators, the running maximum and sum of each row in its lane.  K and V
// come in stages copied HBM -> LDS without registers, one stage ahead.  A
// 32 x 32 block costs two products, S^T = K Q^T and O^T += V^T P^T, with P
// straight from the accumulators; a block of which a wave sees nothing is
// skipped, one that it sees whole takes no mask.
#include "esa_sink.hpp"

namespace esa {

namespace {

template <int D, Elem E>
struct SinkFwdCfg {
  static constexpr int WAVES_PER_SIMD =
      E == Elem::f32 ? (D >= 128 ? 1 : 2) : D >= 128 ? 2 : 4;
};

template <int D, Elem E>
__global__ __launch_bounds__(256, (SinkFwdCfg<D, E>::WAVES_PER_SIMD)) void sink_fwd_kernel(
    SinkArgs A) {
  using T = SinkTile<D, E>;
  using Stage = SinkStage<D, E, 32, 256>;
  using LdsT = typename T::LdsT;
  constexpr int ND = T::ND, N = 32 * D;
  // four stages of 32 keys; separate objects, so that reads of one are seen
  // not to depend on the copies into another
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
  const KeyStages keys = key_stages<32>(A, si, r0, sink_end);

  const int tid = threadIdx.x;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hf = lane >> 5;
  const int r = r0 + wave * 32 + l32;
  const bool row_in = r < A.q_len;
  const int p = si.base + r;
  const int pb = keys.pb, pw0 = si.base + r0 + wave * 32, pw1 = min(pw0 + 31, pb);
  const int n_all = keys.n_all;
  const WaveStages ws = wave_stages<32>(keys, pw0, pw1, W, sink_end);

  T t;
  t.init(lane);
  typename T::Frag qf;
  t.load_frag(qf, (const char*)A.q + ((int64_t)b * A.qsb + (int64_t)h * A.qsh +
                                      (int64_t)r * A.qss) * T::ES, row_in, A.d_real);
  f32x16 oacc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) oacc[d] = f32x16{};
  float m_run = -INFINITY, l_run = 0.f, n_run = 0.f;
  const float scale = A.scale_log2;

  Stage ks, vs;
  ks.init((const char*)A.k + ((int64_t)b * A.ksb + (int64_t)kvh * A.ksh) * T::ES, A.kss,
          A.kv_len, A.d_real, tid);
  vs.init((const char*)A.v + ((int64_t)b * A.vsb + (int64_t)kvh * A.vsh) * T::ES, A.vss,
          A.kv_len, A.d_real, tid);

  // Stages run as a pipeline: while a stage's scores go through the softmax
  // and its product with V, the next stage's scores are formed, so the matrix
  // pipe has work beside the exponentials.  s: the coming stage's scores (of
  // the keys that the wave sees), top: each row's largest of them; used: the
  // wave sees some of its keys.
  f32x16 s = f32x16{};
  float top = -INFINITY;
  bool used = false;
  auto row_top = [&](const f32x16& x) __attribute__((always_inline)) {
    float y = fmaxf(x[0], x[1]);
#pragma unroll
    for (int i = 2; i < 16; ++i) y = fmaxf(y, x[i]);
    return y;
  };
  auto hide = [&](f32x16& x, float& y, int i) __attribute__((always_inline)) {
    if (!ws.full(i)) {
      const int k0 = keys.key0(i);
      uint32_t m[16];
      key_masks<0>(m, seen_keys(p, k0, W, sink_end) >> (4 * hf));
      mask_select(x, m);
      y = row_top(x);
    }
  };
  // stage i: its V in vbuf, the next stage's K in kbuf
  auto step = [&](const LdsT* vbuf, const LdsT* kbuf, int i) __attribute__((always_inline)) {
    const bool next = ws.sees(i + 1);
    f32x16 sn = f32x16{};
    if (!used) {
      if (next) {
        t.row_product(sn, kbuf, 0, qf);
        top = row_top(sn);
        hide(sn, top, i + 1);
        s = sn;
      }
      used = next;
      return;
    }
    top = half_max(top);
    float m_use = m_run == -INFINITY ? 0.f : m_run;
    // the running maximum rises only past the slack (or at a row's first
    // visible key)
    const float over = __builtin_fmaf(top, scale, -m_use);
    const bool grow = over > (m_run == -INFINITY ? -INFINITY : kRescaleSlack);
    if (wave_any(grow)) {
      const float m_new = grow ? m_use + over : m_run;
      const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
      l_run *= alpha;
      n_run *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d) oacc[d] *= alpha;
      m_run = m_new;
      m_use = m_run == -INFINITY ? 0.f : m_run;
    }
    // (past the wave's last key the product is of whatever the buffer holds,
    // and dropped: no branch splits the scores from the softmax)
    if constexpr (T::ES == 2) {
      // in written order: products and exponentials side by side, V's reads
      // ahead of the products that take them
      typename T::V8 ka[T::NS];
#pragma unroll
      for (int k = 0; k < T::NS; ++k) ka[k] = t.row_operand(kbuf, 0, k);
      u32x4 va[ND][2];
      typename T::P pp;
      auto exps = [&](int q) __attribute__((always_inline)) {  // two of the 16
        s[2 * q] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * q], scale, -m_use));
        s[2 * q + 1] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * q + 1], scale, -m_use));
        l_run += s[2 * q] + s[2 * q + 1];
        asm volatile("" : "+v"(l_run));  // summed here, not behind the last product
        pp.w[q] = T::M::pack2(s[2 * q], s[2 * q + 1]);
      };
      constexpr int H = T::NS / 2, EH = 4 / H > 0 ? 4 / H : 1;  // exponential pairs a product
#pragma unroll
      for (int k = 0; k < H; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        sn = T::M::mfma32(ka[k], qf.f[k], sn);
        if (k < ND) va[k][0] = t.col_operand(vbuf, 0, k, 0);
#pragma unroll
        for (int e = 0; e < EH; ++e) exps(k * EH + e);
      }
#pragma unroll
      for (int k = 0; k < H; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        sn = T::M::mfma32(ka[H + k], qf.f[H + k], sn);
        if (k < ND) va[k][1] = t.col_operand(vbuf, 0, k, 1);
#pragma unroll
        for (int e = 0; e < EH; ++e) {
          exps(4 + k * EH + e);
          if (e == 0 && k < ND) t.col_step(oacc[k], va[k][0], pp, 0);
        }
      }
      // O is normalised by the probabilities that its product used
#pragma unroll
      for (int k = 0; k < ND; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        t.col_step(oacc[k], va[k][1], pp, 1);
        n_run = T::M::dot2(pp.w[2 * k], n_run);
        n_run = T::M::dot2(pp.w[2 * k + 1], n_run);
        if (ND == 2) {
          n_run = T::M::dot2(pp.w[2 * k + 4], n_run);
          n_run = T::M::dot2(pp.w[2 * k + 5], n_run);
        }
        asm volatile("" : "+v"(n_run));
      }
      top = row_top(sn);
      __builtin_amdgcn_sched_barrier(0);
    } else {
      t.row_product(sn, kbuf, 0, qf);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        s[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k], scale, -m_use));
        l_run += s[k];
      }
      n_run = l_run;
      t.col_product(oacc, vbuf, 0, t.pack(s));
      top = row_top(sn);
    }
    if (next) hide(sn, top, i + 1);
    s = sn;
    used = next;
  };
  // stage i's wait: its own loads and the next stage's have landed for every
  // wave; the one after may be on its way
  auto ready = [&](int i) __attribute__((always_inline)) {
    if (i + 2 < n_all)
      stage_wait<2 * Stage::LOADS>();
    else
      stage_wait<0>();
  };
  auto issue = [&](int i, LdsT* kd, LdsT* vd) __attribute__((always_inline)) {
    if (i < n_all) {
      ks.issue(keys.key0(i), kd, wave);
      vs.issue(keys.key0(i), vd, wave);
    }
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
      top = row_top(s);
      hide(s, top, 0);
      used = true;
    }
  }
  for (int i = 0; i < n_all; i += 4) {
    ready(i);
    issue(i + 3, k3_, v3_);
    step(v0_, k1_, i);
    if (i + 1 >= n_all) break;
    ready(i + 1);
    issue(i + 4, k0_, v0_);
    step(v1_, k2_, i + 1);
    if (i + 2 >= n_all) break;
    ready(i + 2);
    issue(i + 5, k1_, v1_);
    step(v2_, k3_, i + 2);
    if (i + 3 >= n_all) break;
    ready(i + 3);
    issue(i + 6, k2_, v2_);
    step(v3_, k0_, i + 3);
  }

  // ---- O rows and log-sum-exp
  const bool met = row_in && !(sum_finite(oacc) && __builtin_isfinite(l_run));
  const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
  const float n_tot = n_run + __shfl_xor(n_run, 32, 64);
  // a row that sees no key (before the sequence's first one): 0 and -inf; one
  // without a place in the cache: NaN
  const bool valid = row_in && row_valid(A, si, b, r);
  float inv = 1.f / n_tot, lse = (m_run + __log2f(l_tot)) * 0.69314718055994530942f;
  if (p < f) {
    inv = 0.f;
    lse = -INFINITY;
  }
  if (!valid) inv = lse = __builtin_nanf("");
  const int64_t orow = (int64_t)b * A.osb + (int64_t)h * A.osh + (int64_t)r * A.oss;
#pragma unroll
  for (int d = 0; d < ND; ++d) store_out32<D, E>(A, orow, 32 * d, oacc[d], inv, hf, row_in);
  if (row_in && A.lse && hf == 0) A.lse[(int64_t)b * A.lsb + (int64_t)h * A.lsh + r] = lse;
  // ---- rows that met a non-finite value, again from their own keys
  uint64_t bad = __builtin_amdgcn_ballot_w64(met);
  bad = (bad | bad >> 32) & 0xffffffffull;
  if (bad) __builtin_amdgcn_s_waitcnt(0);  // the stores above come first
  while (bad) {
    const int i = __builtin_ctzll(bad);
    bad &= bad - 1;
    const int row = r0 + wave * 32 + i;
    if (row_valid(A, si, b, row)) fix_row<E>(A, b, h, kvh, row, si.base + row, f, sink_end, lane);
  }
}

template <Elem E>
void launch_elem(const SinkArgs& a, hipStream_t stream) {
  const int64_t grid = (int64_t)a.B * a.H * a.nqb;
  SinkArgs g = a;
  g.xcd_runs = sink_xcd_runs(a, grid);
  if (a.d_real <= 64)
    sink_fwd_kernel<64, E><<<(unsigned)grid, 256, 0, stream>>>(g);
  else
    sink_fwd_kernel<128, E><<<(unsigned)grid, 256, 0, stream>>>(g);
}

}  // namespace

hipError_t launch_sink_fwd(const SinkArgs& a, hipStream_t stream) {
  (void)hipGetLastError();
  if (a.elem == (int)Elem::f32)
    launch_elem<Elem::f32>(a, stream);
  else if (a.elem == (int)Elem::bf16)
    launch_elem<Elem::bf16>(a, stream);
  else
    launch_elem<Elem::f16>(a, stream);
  return hipGetLastError();
}

}  // namespace esa
