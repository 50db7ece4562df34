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
  static constexpr int STAGE = E == Elem::f32 ? 32 : 64;  // keys
  static constexpr int NB = STAGE / 32;
  static constexpr int WAVES_PER_SIMD = E == Elem::f32 ? 1 : 2;
};

template <int D, Elem E>
__global__ __launch_bounds__(256, (SinkFwdCfg<D, E>::WAVES_PER_SIMD)) void sink_fwd_kernel(
    SinkArgs A) {
  using C = SinkFwdCfg<D, E>;
  using T = SinkTile<D, E>;
  using Stage = SinkStage<D, E, C::STAGE, 256>;
  using LdsT = typename T::LdsT;
  constexpr int ND = T::ND;
  // separate objects, so that reads of one buffer are seen not to depend on
  // the copies into the other
  __shared__ __attribute__((aligned(1024))) LdsT k_st0[C::STAGE * D];
  __shared__ __attribute__((aligned(1024))) LdsT v_st0[C::STAGE * D];
  __shared__ __attribute__((aligned(1024))) LdsT k_st1[C::STAGE * D];
  __shared__ __attribute__((aligned(1024))) LdsT v_st1[C::STAGE * D];

  const RowItem it = row_item(A);
  const int b = it.b, h = it.h, kvh = it.kvh, r0 = it.qb * 128;
  const SeqInfo si = seq_info(A, b);
  const int f = si.first, sink_end = min(f + A.sinks, A.kv_len), W = A.window;
  const KeyStages keys = key_stages<C::STAGE>(A, si, r0, sink_end);

  const int tid = threadIdx.x;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hf = lane >> 5;
  const int r = r0 + wave * 32 + l32;
  const bool row_in = r < A.q_len;
  const int p = si.base + r;
  const int pb = keys.pb, pw0 = si.base + r0 + wave * 32, pw1 = min(pw0 + 31, pb);
  const int n_all = keys.n_all;

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

  auto block = [&](const LdsT* kbuf, const LdsT* vbuf, int kb, int k0)
                   __attribute__((always_inline)) {
    if (pw0 > pb || none_seen(pw0, pw1, k0, W, sink_end)) return;
    const bool full = all_seen(pw0, pw0 + 31, k0, W, sink_end);
    f32x16 s = f32x16{};
    if (!full) mask_init<0>(s, ~(seen_keys(p, k0, W, sink_end) >> (4 * hf)));
    t.row_product(s, kbuf, kb, qf);
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    float smax = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_fmaf(s[i], scale, -m_use);
      smax = fmaxf(smax, s[i]);
    }
    smax = half_max(smax);
    // the running maximum rises only past the slack (or at a row's first
    // visible key)
    const float thr = m_run == -INFINITY ? -INFINITY : kRescaleSlack;
    const bool grow = smax > thr;
    if (wave_any(grow)) {
      const float delta = grow ? smax : 0.f;
      const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - (m_use + delta)) : 1.0f;
      l_run *= alpha;
      n_run *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d) oacc[d] *= alpha;
      m_run = grow ? m_use + delta : m_run;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] -= delta;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(s[i]);
      l_run += s[i];
    }
    const typename T::P pp = t.pack(s);
    // O is normalised by the probabilities that its product used
    n_run = T::psum(pp, n_run);
    t.col_product(oacc, vbuf, kb, pp);
  };
  auto stage = [&](const LdsT* kbuf, const LdsT* vbuf, int i) __attribute__((always_inline)) {
    const int k0 = keys.key0(i);
#pragma unroll
    for (int kb = 0; kb < C::NB; ++kb) block(kbuf, vbuf, kb, k0 + 32 * kb);
  };
  if (n_all > 0) {
    ks.issue(keys.key0(0), k_st0, wave);
    vs.issue(keys.key0(0), v_st0, wave);
  }
  for (int i = 0; i < n_all; i += 2) {
    stage_ready();
    if (i + 1 < n_all) {
      ks.issue(keys.key0(i + 1), k_st1, wave);
      vs.issue(keys.key0(i + 1), v_st1, wave);
    }
    stage(k_st0, v_st0, i);
    if (i + 1 >= n_all) break;
    stage_ready();
    if (i + 2 < n_all) {
      ks.issue(keys.key0(i + 2), k_st0, wave);
      vs.issue(keys.key0(i + 2), v_st0, wave);
    }
    stage(k_st1, v_st1, i + 1);
  }

  // ---- O rows and log-sum-exp
  const bool met = row_in && !(sum_finite(oacc) && __builtin_isfinite(l_run));
  const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
  const float n_tot = n_run + __shfl_xor(n_run, 32, 64);
  if (row_in) {
    // a row that sees no key (before the sequence's first one): 0 and -inf;
    // one without a place in the cache: NaN
    const bool valid = row_valid(A, si, b, r);
    float inv = 1.f / n_tot, lse = (m_run + __log2f(l_tot)) * 0.69314718055994530942f;
    if (p < f) {
      inv = 0.f;
      lse = -INFINITY;
    }
    if (!valid) inv = lse = __builtin_nanf("");
    char* orow = (char*)A.o + ((int64_t)b * A.osb + (int64_t)h * A.osh + (int64_t)r * A.oss) *
                                  T::ES;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int dim = 32 * d + 8 * q4 + 4 * hf;
        if (dim < A.d_real)
          T::store4(orow, dim, oacc[d][4 * q4] * inv, oacc[d][4 * q4 + 1] * inv,
                    oacc[d][4 * q4 + 2] * inv, oacc[d][4 * q4 + 3] * inv);
      }
    if (A.lse && hf == 0) A.lse[(int64_t)b * A.lsb + (int64_t)h * A.lsh + r] = lse;
  }
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
