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
// read and dx written).  A workgroup takes a tile of up to eight tokens, forms
// their cosines and sines once in LDS (one float64 product and one sincospi
// per pair and token, shared by all heads), then streams the rows of every
// head: LPR lanes of a wave hold a row, V elements each (16 bytes, or 8 where
// a pair's halves do not start on 16-byte pieces), and a pair's other half
// comes from its lane by a shuffle.  Tables of cosines would be read from HBM
// per token; here nothing but the frequencies is.
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

template <Elem E, int V, int LPR, int MODE>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs A) {
  using T = typename ElemT<E>::T;
  constexpr int RPP = 256 / LPR;  // rows a pass
  __shared__ float2 cs[kRotaryTokens * 128];
  __shared__ int64_t slot[kRotaryTokens];  // append: cache row, or -1

  const int tid = threadIdx.x;
  const int lane = tid % LPR, sub = tid / LPR;
  const int e0 = lane * V;
  const bool on = e0 < A.D;
  const int half = A.rd / 2;
  // this lane's part in the rotation: first element's pair, its partner lane
  // and the sign of the partner's product (pairs of halves)
  const bool rot = e0 < A.rd;
  const bool second = !A.interleaved && e0 >= half;
  const int pair0 = A.interleaved ? e0 / 2 : second ? e0 - half : e0;
  const int partner = (tid & 63) + (rot && !A.interleaved ? (second ? -half / V : half / V) : 0);
  const float sign = second ? 1.f : -1.f;

  float wq[V], wk[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    wq[e] = on && A.wq ? load_gain(A.wq, A.welem, e0 + e) : 1.f;
    wk[e] = on && A.wk ? load_gain(A.wk, A.welem, e0 + e) : 1.f;
  }
  float gq[V], gk[V];  // backward: sums of g * n
#pragma unroll
  for (int e = 0; e < V; ++e) gq[e] = gk[e] = 0.f;

  const int h0 = blockIdx.y * A.heads_per_split;
  const int nh = min(A.heads_per_split, A.heads - h0);
  const float inv_d = 1.f / (float)A.D;

  for (int tile = blockIdx.x; tile < A.n_tiles; tile += gridDim.x) {
    const int b = (int)fast_div((uint32_t)tile, A.div_tiles);
    const int t0 = (tile - b * A.tiles_per_seq) << A.log_t;
    const int nt = min(1 << A.log_t, A.n - t0);
    const int64_t* pos = A.pos + (int64_t)b * A.pos_sb;
    if (tile != (int)blockIdx.x) __syncthreads();  // the previous tile's reads of cs
    int64_t base = 0;
    if constexpr (MODE == kAppend) {
      base = pos[0];
      base += base < 0 ? A.kv_len : 0;
    }
    for (int i = tid; i < nt * half; i += 256) {
      const int t = (int)fast_div((uint32_t)i, A.div_half), f = i - t * half;
      int64_t p = pos[t0 + t];
      if constexpr (MODE == kAppend) p += p < 0 ? A.kv_len : 0;
      double turns = (double)p * A.inv_freq[f] * 0.15915494309189533577;
      turns -= rint(turns);
      float s, c;
      sincospif(2.f * (float)turns, &s, &c);
      cs[i] = make_float2(c, s);
    }
    if constexpr (MODE == kAppend) {
      // row s of the sequence belongs at base + s inside the cache; any other
      // position (out of range, repeated, out of order) is written nowhere
      if (tid < nt) {
        int64_t p = pos[t0 + tid];
        p += p < 0 ? A.kv_len : 0;
        slot[tid] = base >= 0 && p == base + t0 + tid && p < A.kv_len ? p : -1;
      }
    }
    __syncthreads();

    const int rows = nt * nh;
    for (int row = sub; row < rows; row += RPP) {
      // heads are the fast axis where a token's heads lie next to each other
      int t, hh;
      if (A.heads_fast) {
        t = (int)fast_div((uint32_t)row, A.div_heads);
        hh = row - t * nh;
        if (nh != A.heads_per_split) {  // the last split's shorter rows
          t = row / nh;
          hh = row - t * nh;
        }
      } else if (nt == 1 << A.log_t) {
        hh = row >> A.log_t;
        t = row - (hh << A.log_t);
      } else {
        hh = row / nt;
        t = row - hh * nt;
      }
      hh += h0;
      const int64_t s = t0 + t;
      int64_t os = s;  // the output's row
      if constexpr (MODE == kAppend) os = slot[t];
      const int kind = hh < A.H ? 0 : hh < A.H + A.Hkv ? 1 : 2;
      const int h = kind == 0 ? hh : hh - A.H - (kind == 2 ? A.Hkv : 0);

      const T* src = kind == 0 ? (const T*)A.q + b * A.qsb + h * A.qsh + s * A.qss
                   : kind == 1 ? (const T*)A.k + b * A.ksb + h * A.ksh + s * A.kss
                               : (const T*)A.v + b * A.vsb + h * A.vsh + s * A.vss;
      Piece<E, V> in;
      in.w = decltype(in.w){};
      if (on) in.w = *(const decltype(in.w)*)(src + e0);
      if constexpr (MODE == kAppend) {
        if (kind == 2) {  // values go to their cache as they are
          if (on && os >= 0)
            *(decltype(in.w)*)((T*)A.vo + b * A.vosb + h * A.vosh + os * A.voss + e0) = in.w;
          continue;
        }
      }
      float x[V], ss = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x[e] = in.get(e);
        ss = __builtin_fmaf(x[e], x[e], ss);
      }
      const float2* crow = cs + t * half;

      if constexpr (MODE != kBwd) {
#pragma unroll
        for (int off = LPR / 2; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, 64);
        const float r = 1.f / sqrtf(__builtin_fmaf(ss, inv_d, A.eps));
        float y[V];
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] *= r * (kind == 0 ? wq[e] : wk[e]);
        if (A.interleaved) {
#pragma unroll
          for (int e = 0; e < V; e += 2) {
            const float2 c = rot ? crow[pair0 + e / 2] : make_float2(1.f, 0.f);
            y[e] = x[e] * c.x - x[e + 1] * c.y;
            y[e + 1] = x[e + 1] * c.x + x[e] * c.y;
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float2 c = rot ? crow[pair0 + e] : make_float2(1.f, 0.f);
            y[e] = x[e] * c.x + sign * __shfl(x[e], partner, 64) * c.y;
          }
        }
        if constexpr (MODE == kAppend) {
          if (os < 0) {
            if (kind == 1) continue;
            // a query row with no place in the cache: NaN, as the attention
            // over the cache gives it
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = __builtin_nanf("");
            os = s;
          }
          if (kind == 0) os = s;
        }
        if (on) {
          T* dst = kind == 0 ? (T*)A.qo + b * A.qosb + h * A.qosh + os * A.qoss
                             : (T*)A.ko + b * A.kosb + h * A.kosh + os * A.koss;
          store_piece<E, V>(dst + e0, y);
        }
      } else {
        const T* gsrc = kind == 0 ? (const T*)A.gq + b * A.gqsb + h * A.gqsh + s * A.gqss
                                  : (const T*)A.gk + b * A.gksb + h * A.gksh + s * A.gkss;
        Piece<E, V> gin;
        gin.w = decltype(gin.w){};
        if (on) gin.w = *(const decltype(gin.w)*)(gsrc + e0);
        float g[V], y[V], dot = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) g[e] = gin.get(e);
        // the rotation undone
        if (A.interleaved) {
#pragma unroll
          for (int e = 0; e < V; e += 2) {
            const float2 c = rot ? crow[pair0 + e / 2] : make_float2(1.f, 0.f);
            y[e] = g[e] * c.x + g[e + 1] * c.y;
            y[e + 1] = g[e + 1] * c.x - g[e] * c.y;
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float2 c = rot ? crow[pair0 + e] : make_float2(1.f, 0.f);
            y[e] = g[e] * c.x - sign * __shfl(g[e], partner, 64) * c.y;
          }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          g[e] = y[e] * (kind == 0 ? wq[e] : wk[e]);
          dot = __builtin_fmaf(g[e], x[e], dot);
        }
#pragma unroll
        for (int off = LPR / 2; off >= 1; off >>= 1) {
          ss += __shfl_xor(ss, off, 64);
          dot += __shfl_xor(dot, off, 64);
        }
        const float r = 1.f / sqrtf(__builtin_fmaf(ss, inv_d, A.eps));
        const float m = dot * inv_d * r * r;  // mean(g gain n) r
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float gn = y[e] * (x[e] * r);
          if (kind == 0) gq[e] += gn; else gk[e] += gn;
          g[e] = r * (g[e] - x[e] * m);
        }
        if (on) {
          T* dst = kind == 0 ? (T*)A.qo + b * A.qosb + h * A.qosh + s * A.qoss
                             : (T*)A.ko + b * A.kosb + h * A.kosh + s * A.koss;
          store_piece<E, V>(dst + e0, g);
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
      for (int e = 0; e < V; ++e) red[sub * (LPR * V) + e0 + e] = which ? gk[e] : gq[e];
      __syncthreads();
      for (int d = tid; d < A.D; d += 256) {
        float sum = 0.f;
        for (int i = 0; i < RPP; ++i) sum += red[i * (LPR * V) + d];
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

template <Elem E, int V, int MODE>
void launch_lpr(const RotaryArgs& a, dim3 grid, hipStream_t stream) {
  const int lanes = (a.D + V - 1) / V;
  if (lanes <= 8)
    rotary_kernel<E, V, 8, MODE><<<grid, 256, 0, stream>>>(a);
  else if (lanes <= 16)
    rotary_kernel<E, V, 16, MODE><<<grid, 256, 0, stream>>>(a);
  else if (lanes <= 32)
    rotary_kernel<E, V, 32, MODE><<<grid, 256, 0, stream>>>(a);
  else
    rotary_kernel<E, V, 64, MODE><<<grid, 256, 0, stream>>>(a);
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
