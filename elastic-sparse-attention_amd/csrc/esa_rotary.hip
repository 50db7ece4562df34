// Norm of each head's queries and keys with their position rotation (gfx950):
// the rows an attention layer reads, or writes into its caches.
//
//   n = x * r,  r = 1 / sqrt(mean(x^2) + eps)      over one head's D elements
//   y = R(p) (n * gain)                            gain shared by the heads
//
// R(p) turns pair i of the first rotary_dim elements by the angle
// p * inv_freq[i]; a pair is elements (i, i + rotary_dim / 2), or (2 i, 2 i + 1)
// interleaved.  Angles are formed and reduced to one turn in float64: in
// float32 the angle of a position past 2^17 is off by 1e-2.  Everything else
// is float32, rounded once when it is stored.  Backward, with g = R(-p) dy:
//
//   dgain = sum over rows of g * n,   dx = r (g gain - n mean(g gain n))
//
// Bound: HBM (each row is read and written once; in the backward x and dy are
// read and dx written), and next to it the instructions a row takes.  LPR
// lanes of a wave hold a row, V elements each (16 bytes, or 8 where a pair's
// halves do not start on 16-byte pieces), and keep to one token: its cosines
// and sines are formed once in LDS (one float64 product and one sincospi a
// pair, shared by all heads; tables would be read from HBM) and stay in
// registers while the lanes go through its heads, the next head's row on its
// way.  A pair's other half comes from its lane by a DPP rotation (16 lanes a
// row) or a shuffle.  Rows past the last-level cache whose heads are side by side
// are taken two heads at a time (SIDE).  32768 tokens of 32 + 8 heads of 128,
// bf16, views of one projection: 158 us, 4.25 TB/s (a copy of as much: 137 us at
// 4.89; 171 with one head at a time; 187 with a row's lanes going from token to
// token of one head, tables read again for each); 15003 tokens of 16 + 4 heads of
// 96, f16: forward 26 (41), backward 45 (58).
#include "esa_rotary.hpp"
#include "esa_mma.hpp"

namespace esa {

namespace {

enum { kFwd = 0, kAppend = 1, kBwd = 2 };

template <Elem E, int V>
struct Piece;
template <>
struct Piece<Elem::f32, 4> {
  u32x4 w;
  __device__ __forceinline__ float get(int e) const { return __uint_as_float(w[e]); }
  __device__ __forceinline__ void set(int e, float x) { w[e] = __float_as_uint(x); }
};
template <Elem E>
struct Piece<E, 8> {
  u32x4 w;
  __device__ __forceinline__ float get(int e) const {
    return MmaT<E>::val((w[e / 2] >> (16 * (e & 1))) & 0xffffu);
  }
  __device__ __forceinline__ void set2(int q, float a, float b) { w[q] = MmaT<E>::pack2(a, b); }
};
template <Elem E>
struct Piece<E, 4> {
  u32x2 w;
  __device__ __forceinline__ float get(int e) const {
    return MmaT<E>::val((w[e / 2] >> (16 * (e & 1))) & 0xffffu);
  }
  __device__ __forceinline__ void set2(int q, float a, float b) { w[q] = MmaT<E>::pack2(a, b); }
};

template <Elem E, int V>
__device__ __forceinline__ void store_piece(typename ElemT<E>::T* p, const float (&y)[V]) {
  Piece<E, V> o;
  if constexpr (E == Elem::f32) {
#pragma unroll
    for (int e = 0; e < V; ++e) o.set(e, y[e]);
  } else {
#pragma unroll
    for (int q = 0; q < V / 2; ++q) o.set2(q, y[2 * q], y[2 * q + 1]);
  }
  *(decltype(o.w)*)p = o.w;
}

__device__ __forceinline__ float load_gain(const void* w, int elem, int i) {
  if (elem == (int)Elem::f32) return ((const float*)w)[i];
  const uint16_t b = ((const uint16_t*)w)[i];
  return elem == (int)Elem::bf16 ? ElemT<Elem::bf16>::load(&b) : ElemT<Elem::f16>::load(&b);
}

__device__ __forceinline__ void store_gain(void* w, int elem, int i, float x) {
  if (elem == (int)Elem::f32)
    ((float*)w)[i] = x;
  else if (elem == (int)Elem::bf16)
    ElemT<Elem::bf16>::store((uint16_t*)w + i, x);
  else
    ElemT<Elem::f16>::store((uint16_t*)w + i, x);
}

// x of the lane that holds the other halves of this lane's pairs
template <int LPR>
__device__ __forceinline__ float other_half(float x, int partner, bool across8) {
  if (LPR == 16 && across8) {
    // lane l ^ 8: a rotation by 8 in each row of 16 lanes
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(
        0, (int)__float_as_uint(x), 0x128, 0xf, 0xf, true));
  }
  return __shfl(x, partner, 64);
}

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int off = LPR / 2; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// SIDE: heads of a token that lane groups take side by side (1, or 2)
template <Elem E, int V, int LPR, int MODE, int SIDE>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs A) {
  using T = typename ElemT<E>::T;
  using P = Piece<E, V>;
  using W = decltype(P::w);
  constexpr int TOK = 256 / LPR;  // tokens of a tile
  __shared__ float2 cs[TOK * (LPR * V / 2)];

  const int tid = threadIdx.x;
  const int lane = tid % LPR, group = tid / LPR;
  const int hsub = group % SIDE;  // the group's heads: hsub + SIDE i
  const int e0 = lane * V;
  const bool on = e0 < A.D;
  const int half = A.rd / 2;
  // this lane's part in the rotation: first element's pair, its partner lane
  const bool rot = e0 < A.rd;
  const bool second = !A.interleaved && e0 >= half;
  const int pair0 = A.interleaved ? e0 / 2 : second ? e0 - half : e0;
  const int partner = (tid & 63) + (rot && !A.interleaved ? (second ? -half / V : half / V) : 0);
  const bool across8 = half == 8 * V;  // (lanes past rd take the value and multiply it by 0)

  float wq[V], wk[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    wq[e] = on && A.wq ? load_gain(A.wq, A.welem, e0 + e) : 1.f;
    wk[e] = on && A.wk ? load_gain(A.wk, A.welem, e0 + e) : 1.f;
  }
  float gq[V], gk[V];  // backward: sums of g * n
#pragma unroll
  for (int e = 0; e < V; ++e) gq[e] = gk[e] = 0.f;

  // this workgroup's heads among q's, k's and (append) v's
  const int h0 = blockIdx.y * A.heads_per_split;
  const int h1 = min(h0 + A.heads_per_split, A.heads);
  const float inv_d = 1.f / (float)A.D;

  for (int tile = blockIdx.x; tile < A.n_tiles; tile += gridDim.x) {
    const int g0 = tile * TOK, nt = min(TOK, A.tokens - g0);
    if (tile != (int)blockIdx.x) __syncthreads();  // the previous tile's reads of cs
    for (int i = tid; i < nt * half; i += 256) {
      const int t = (int)fast_div((uint32_t)i, A.div_half), f = i - t * half;
      const int b = (int)fast_div((uint32_t)(g0 + t), A.div_n);
      int64_t p = A.pos[(int64_t)b * A.pos_sb + (g0 + t - b * A.n)];
      if constexpr (MODE == kAppend) p += p < 0 ? A.kv_len : 0;
      double turns = (double)p * A.inv_freq[f] * 0.15915494309189533577;
      turns -= rint(turns);
      float s, c;
      sincospif(2.f * (float)turns, &s, &c);
      cs[i] = make_float2(c, s);
    }
    __syncthreads();
    // (no barrier before the next tile's first one)
#pragma unroll 1
    for (int sub = group / SIDE; sub < nt; sub += TOK / SIDE) {
      const int64_t b = fast_div((uint32_t)(g0 + sub), A.div_n), s = g0 + sub - b * A.n;
      int64_t os = s;  // the output's row
      if constexpr (MODE == kAppend) {
        // row s of the sequence belongs at base + s inside the cache; any other
        // position (out of range, repeated, out of order) is written nowhere
        const int64_t* pos = A.pos + b * A.pos_sb;
        int64_t base = pos[0], p = pos[s];
        base += base < 0 ? A.kv_len : 0;
        p += p < 0 ? A.kv_len : 0;
        os = base >= 0 && p == base + s && p < A.kv_len ? p : -1;
      }
      // y[e] = x[e] c[e] + (the pair's other element) sn[e]
      float c[V], sn[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float2 t = make_float2(1.f, 0.f);
        if (rot) t = cs[sub * half + pair0 + (A.interleaved ? e / 2 : e)];
        c[e] = t.x;
        sn[e] = (A.interleaved ? e & 1 : second) ? t.y : -t.y;
      }
      auto turn = [&](const float (&x)[V], float (&y)[V], float dir) __attribute__((always_inline)) {
        if (A.interleaved) {
#pragma unroll
          for (int e = 0; e < V; ++e) y[e] = x[e] * c[e] + dir * x[e ^ 1] * sn[e];
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            y[e] = x[e] * c[e] + dir * other_half<LPR>(x[e], partner, across8) * sn[e];
        }
        // (elements past rotary_dim as they are: a neighbour's infinity is not theirs)
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = rot ? y[e] : x[e];
      };
      // the group's of `n` heads of q or k from src (and g), results to dst
      auto heads = [&](const T* src, int64_t sh, const T* g, int64_t gh, T* dst, int64_t dh,
                       int n, const float (&w)[V], float (&sums)[V], bool lost)
                       __attribute__((always_inline)) {
        const int count = (n - hsub + SIDE - 1) / SIDE;
        if (SIDE > 1) {
          if (count <= 0) return;
          src += hsub * sh;
          g += hsub * gh;
          dst += hsub * dh;
          sh *= SIDE;
          gh *= SIDE;
          dh *= SIDE;
        }
        P in, gin;
        in.w = gin.w = W{};
        if (on) in.w = *(const W*)src;
        if (MODE == kBwd && on) gin.w = *(const W*)g;
        for (int i = 0; i < count; ++i) {
          const P xin = in, ggin = gin;
          src += sh;
          g += gh;
          if (i + 1 < count && on) {  // the next head's row, on its way meanwhile
            in.w = *(const W*)src;
            if (MODE == kBwd) gin.w = *(const W*)g;
          }
          float x[V], y[V], ss = 0.f;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            x[e] = xin.get(e);
            ss = __builtin_fmaf(x[e], x[e], ss);
          }
          if constexpr (MODE != kBwd) {
            const float r = rsqrtf(__builtin_fmaf(row_sum<LPR>(ss), inv_d, A.eps));
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] *= r * w[e];
            turn(x, y, 1.f);
            if (MODE == kAppend && lost) {
#pragma unroll
              for (int e = 0; e < V; ++e) y[e] = __builtin_nanf("");
            }
          } else {
            float gr[V], dot = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) gr[e] = ggin.get(e);
            turn(gr, y, -1.f);  // the rotation undone
#pragma unroll
            for (int e = 0; e < V; ++e) {
              gr[e] = y[e] * w[e];
              dot = __builtin_fmaf(gr[e], x[e], dot);
            }
            ss = row_sum<LPR>(ss);
            dot = row_sum<LPR>(dot);
            const float r = rsqrtf(__builtin_fmaf(ss, inv_d, A.eps));
            const float m = dot * inv_d * r * r;  // mean(g gain n) r
#pragma unroll
            for (int e = 0; e < V; ++e) {
              sums[e] += y[e] * (x[e] * r);
              y[e] = r * (gr[e] - x[e] * m);
            }
          }
          if (on) store_piece<E, V>(dst, y);
          dst += dh;
        }
      };
      const int nq = min(h1, A.H) - h0;
      if (nq > 0)
        heads((const T*)A.q + b * A.qsb + h0 * A.qsh + s * A.qss + e0, A.qsh,
              (const T*)A.gq + b * A.gqsb + h0 * A.gqsh + s * A.gqss + e0, A.gqsh,
              (T*)A.qo + b * A.qosb + h0 * A.qosh + s * A.qoss + e0, A.qosh, nq, wq, gq,
              // a query row with no place in the cache: NaN, as the attention
              // over the cache gives it
              MODE == kAppend && os < 0);
      const int k0 = max(h0 - A.H, 0), nk = min(h1 - A.H, A.Hkv) - k0;
      if (nk > 0 && os >= 0)
        heads((const T*)A.k + b * A.ksb + k0 * A.ksh + s * A.kss + e0, A.ksh,
              (const T*)A.gk + b * A.gksb + k0 * A.gksh + s * A.gkss + e0, A.gksh,
              (T*)A.ko + b * A.kosb + k0 * A.kosh + os * A.koss + e0, A.kosh, nk, wk, gk, false);
      if constexpr (MODE == kAppend) {  // values go to their cache as they are
        const int v0 = max(h0 - A.H - A.Hkv, 0), v1 = h1 - A.H - A.Hkv;
        const T* src = (const T*)A.v + b * A.vsb + (v0 + hsub) * A.vsh + s * A.vss + e0;
        T* dst = (T*)A.vo + b * A.vosb + (v0 + hsub) * A.vosh + os * A.voss + e0;
        for (int h = v0 + hsub; h < v1 && os >= 0 && on; h += SIDE) {
          *(W*)dst = *(const W*)src;
          src += SIDE * A.vsh;
          dst += SIDE * A.vosh;
        }
      }
    }
  }

  if constexpr (MODE == kBwd) {
    // the gains' sums over the workgroup's rows, in the order of its lanes
    if (!A.partial) return;
    __shared__ float red[256 * V];
    float* out = A.partial + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * A.D;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < V; ++e) red[group * (LPR * V) + e0 + e] = which ? gk[e] : gq[e];
      __syncthreads();
      for (int d = tid; d < A.D; d += 256) {
        float sum = 0.f;
        for (int i = 0; i < TOK; ++i) sum += red[i * (LPR * V) + d];
        out[which * A.D + d] = sum;
      }
    }
  }
}

// The workgroups' sums of g * n joined, in a fixed order: eight columns a
// workgroup, 128 lanes to a column.
__global__ __launch_bounds__(1024) void rotary_gain_kernel(const float* partial, int n_parts,
                                                           int cols, int D, void* dwq, void* dwk,
                                                           int welem) {
  __shared__ float red[128][8];
  const int c = threadIdx.x & 7, r = threadIdx.x >> 3;
  const int col = blockIdx.x * 8 + c;
  float sum = 0.f;
  if (col < cols)
    for (int i = r; i < n_parts; i += 128) sum += partial[(int64_t)i * cols + col];
  red[r][c] = sum;
  __syncthreads();
  for (int off = 64; off >= 1; off >>= 1) {
    if (r < off) red[r][c] += red[r + off][c];
    __syncthreads();
  }
  if (r == 0 && col < cols) {
    void* dst = col < D ? dwq : dwk;
    if (dst) store_gain(dst, welem, col < D ? col : col - D, red[0][c]);
  }
}

template <Elem E, int V, int LPR, int MODE>
void launch_side(const RotaryArgs& a, dim3 grid, hipStream_t stream) {
  if constexpr (MODE != kBwd)
    if (a.side == 2) {
      rotary_kernel<E, V, LPR, MODE, 2><<<grid, 256, 0, stream>>>(a);
      return;
    }
  rotary_kernel<E, V, LPR, MODE, 1><<<grid, 256, 0, stream>>>(a);
}

template <Elem E, int V, int MODE>
void launch_lpr(const RotaryArgs& a, dim3 grid, hipStream_t stream) {
  if (a.lanes == 8)
    launch_side<E, V, 8, MODE>(a, grid, stream);
  else if (a.lanes == 16)
    launch_side<E, V, 16, MODE>(a, grid, stream);
  else if (a.lanes == 32)
    launch_side<E, V, 32, MODE>(a, grid, stream);
  else
    launch_side<E, V, 64, MODE>(a, grid, stream);
}

template <int MODE>
void launch_mode(const RotaryArgs& a, dim3 grid, hipStream_t stream) {
  if (a.elem == (int)Elem::f32)
    launch_lpr<Elem::f32, 4, MODE>(a, grid, stream);
  else if (a.elem == (int)Elem::bf16)
    a.vec == 8 ? launch_lpr<Elem::bf16, 8, MODE>(a, grid, stream)
               : launch_lpr<Elem::bf16, 4, MODE>(a, grid, stream);
  else
    a.vec == 8 ? launch_lpr<Elem::f16, 8, MODE>(a, grid, stream)
               : launch_lpr<Elem::f16, 4, MODE>(a, grid, stream);
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& a, int mode, hipStream_t stream) {
  (void)hipGetLastError();
  const dim3 grid((unsigned)a.grid_tiles, (unsigned)a.n_splits);
  if (mode == kFwd)
    launch_mode<kFwd>(a, grid, stream);
  else if (mode == kAppend)
    launch_mode<kAppend>(a, grid, stream);
  else
    launch_mode<kBwd>(a, grid, stream);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || mode != kBwd || !a.partial) return e;
  const int cols = 2 * a.D;
  rotary_gain_kernel<<<(cols + 7) / 8, 1024, 0, stream>>>(
      a.partial, a.grid_tiles * a.n_splits, cols, a.D, a.dwq, a.dwk, a.welem);
  return hipGetLastError();
}

}  // namespace esa
