// Forward of attention over a causal window with sinks (gfx950).
//
//   s = scale q k^T on visible keys,  o = softmax(s) v,  lse = log sum exp(s)
//
// One workgroup (4 waves) takes 128 rows of one (sequence, head) and walks
// the keys they see: the sinks' stages, then the window's, or one run of
// stages where the two meet.  Each wave holds 32 rows: Q in registers, O^T in
// accumulators, the running maximum and sum of each row in its lane.  K and V
// come in stages of 32 keys copied HBM -> LDS without registers, up to two
// stages ahead.  A 32 x 32 block costs two products, S^T = K Q^T and
// O^T += V^T P^T, with P straight from the accumulators; a stage of which a
// wave sees nothing is skipped, one that it sees whole takes no mask.  Where a
// grid leaves CUs idle a block's stages are cut into ranges, a workgroup each,
// that leave (O, m, l) for a join.
//
// Bound: the vector instructions of a block (about 92 beside its 16 matrix
// instructions at head_dim 128; a SIMD's vector and matrix pipes overlap in
// part only: 8 float32 fma after each of two waves' products cost 33% of the
// products' time on top, 4 nothing), so waves are what counts: with registers
// for three a SIMD (168, reads' addresses formed anew, three stages in LDS)
// instead of two, 32768 rows of 32 heads on 8, window 4096, bf16, take 2.11 ms
// (980 TFLOP/s) instead of 2.17 on one card (2.02 on another), though a grid
// that is one round of two blocks a CU gains no wave: 2048 such rows 158 us
// instead of 152.  Operands read 2, 3 or 4 products ahead: 2.03, 2.02, 2.05 ms.
// 8192 rows, window 1024, with o's residual: 180 us; 8 padded sequences of 4099,
// 16 heads of 64, window 500, f16 (four waves): 130 us, against 149 with three.
#include "esa_sink.hpp"

namespace esa {

namespace {

template <int D, Elem E>
struct SinkFwdCfg {
  static constexpr int WAVES_PER_SIMD =
      E == Elem::f32 ? (D >= 128 ? 1 : 2) : D >= 128 ? 3 : 4;
};

template <int D, int DR, Elem E>
__global__ __launch_bounds__(256, (SinkFwdCfg<D, E>::WAVES_PER_SIMD)) void sink_fwd_kernel(
    SinkArgs A) {
  using T = SinkTile<D, E, true, DR>;
  using Stage = SinkStage<D, E, 32, 256>;
  using LdsT = typename T::LdsT;
  constexpr int ND = T::ND, N = 32 * D;
  // three stages of 32 keys; separate objects, so that reads of one are seen
  // not to depend on the copies into another
  __shared__ __attribute__((aligned(1024))) LdsT k0_[N];
  __shared__ __attribute__((aligned(1024))) LdsT v0_[N];
  __shared__ __attribute__((aligned(1024))) LdsT k1_[N];
  __shared__ __attribute__((aligned(1024))) LdsT v1_[N];
  __shared__ __attribute__((aligned(1024))) LdsT k2_[N];
  __shared__ __attribute__((aligned(1024))) LdsT v2_[N];

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
  // this workgroup's range of the stages, from i0 (all of them, unless the grid
  // is small and they are cut)
  const int i0 = (int)((int64_t)keys.n_all * it.split / A.splits);
  const int n_all = (int)((int64_t)keys.n_all * (it.split + 1) / A.splits);
  WaveStages ws = wave_stages(keys, pw0, pw1, W, sink_end);
  ws.last = min(ws.last, n_all - 1);

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
      // In written order, each operand read AHEAD products ahead: the first half
      // of the scores beside the first half of the exponentials, the second half
      // of both beside the first products with V, then V's rest.
      constexpr int AHEAD = 3, NS = T::NS, H = NS / 2;
      typename T::V8 ka[NS];
      u32x4 va[2 * ND];
      typename T::P pp;
      int base, vbase;  // of the reads' addresses
      // product i is of scores (its number) or, from there on, with V
      auto order = [](int i) constexpr {
        return i < H ? i : i >= H + NS ? NS + i - NS : (i - H) % 2 ? NS + (i - H) / 2 : (i + H) / 2;
      };
      auto read = [&](int i) __attribute__((always_inline)) {
        if (i >= 2 * NS) return;
        const int o = order(i), k = o % NS;
        if (o == 0) base = T::fresh(t.ra[0]);
        if (o == NS) vbase = T::fresh(t.ca[0]);
        if (o < NS)
          ka[k] = t.row_operand(kbuf, 0, k, base);
        else
          va[k] = t.col_operand(vbuf, 0, k % ND, k / ND, vbase);
      };
      auto exps = [&](int k) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 8 * k / NS; q < 8 * (k + 1) / NS; ++q) {  // pairs of keys
          s[2 * q] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * q], scale, -m_use));
          s[2 * q + 1] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * q + 1], scale, -m_use));
          l_run += s[2 * q] + s[2 * q + 1];
          pp.w[q] = T::M::pack2(s[2 * q], s[2 * q + 1]);
        }
        asm volatile("" : "+v"(l_run));  // summed here, not behind the last product
      };
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) read(i);
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        const int o = order(i), k = o % NS;
        if (o < NS) {
          sn = T::M::mfma32(ka[k], qf.f[k], sn);
          exps(k);
        } else {
          T::col_step(oacc[k % ND], va[k], pp, k / ND);
          // O is normalised by the probabilities that its product used
#pragma unroll
          for (int w = 4 * (k % ND) / ND; w < 4 * (k % ND + 1) / ND; ++w)
            n_run = T::M::dot2(pp.w[4 * (k / ND) + w], n_run);
          asm volatile("" : "+v"(n_run));
        }
        read(i + AHEAD);
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
  // Stage i's wait, for every wave: its V and the next stage's K have landed
  // (the next V, issued last, may be on its way)
  auto ready = [&](int i) __attribute__((always_inline)) {
    if (i + 1 < n_all)
      stage_wait<Stage::LOADS>();
    else
      stage_wait<0>();
  };
  auto issue = [&](int i, LdsT* kd, LdsT* vd) __attribute__((always_inline)) {
    if (i < n_all) {
      ks.issue(keys.key0(i), kd, wave);
      vs.issue(keys.key0(i), vd, wave);
    }
  };
  issue(i0, k0_, v0_);
  issue(i0 + 1, k1_, v1_);
  if (n_all > i0) {
    if (n_all > i0 + 1)
      stage_wait<3 * Stage::LOADS>();
    else
      stage_wait<0>();
    if (ws.sees(i0)) {
      t.row_product(s, k0_, 0, qf);
      top = row_top(s);
      hide(s, top, i0);
      used = true;
    }
  }
  for (int i = i0; i < n_all; i += 3) {
    ready(i);
    issue(i + 2, k2_, v2_);
    step(v0_, k1_, i);
    if (i + 1 >= n_all) break;
    ready(i + 1);
    issue(i + 3, k0_, v0_);
    step(v1_, k2_, i + 1);
    if (i + 2 >= n_all) break;
    ready(i + 2);
    issue(i + 4, k1_, v1_);
    step(v2_, k0_, i + 2);
  }

  // ---- O rows and log-sum-exp
  const bool met = row_in && !(sum_finite(oacc) && __builtin_isfinite(l_run));
  const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
  const float n_tot = n_run + __shfl_xor(n_run, 32, 64);
  if (A.splits > 1) {  // a part
    const int i = r * A.groups + h - kvh * A.groups;
    const int64_t unit = (((int64_t)(b * A.Hkv + kvh) * A.row_tiles + (i >> 4)) * A.splits +
                          it.split) * 16 + (i & 15);
    if (row_in) {
      float* row = A.partial + unit * D + 4 * hf;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *(f32x4*)(row + 32 * d + 8 * q) = f32x4{oacc[d][4 * q], oacc[d][4 * q + 1],
                                                  oacc[d][4 * q + 2], oacc[d][4 * q + 3]};
      if (hf == 0) {
        float* ml = A.part_ml + unit * 3;
        ml[0] = m_run;
        ml[1] = l_tot;
        ml[2] = n_tot;
      }
    }
    return;
  }
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
  const int64_t grid = (int64_t)a.B * a.H * a.nqb * a.splits;
  SinkArgs g = a;
  g.xcd_runs = sink_xcd_runs(a, grid);
  if (a.d_real <= 64)
    sink_fwd_kernel<64, 64, E><<<(unsigned)grid, 256, 0, stream>>>(g);
  else if (a.d_real <= 96)
    sink_fwd_kernel<128, 96, E><<<(unsigned)grid, 256, 0, stream>>>(g);
  else
    sink_fwd_kernel<128, 128, E><<<(unsigned)grid, 256, 0, stream>>>(g);
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
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || a.splits == 1 ? e : launch_sink_rows_join(a, stream);
}

}  // namespace esa
