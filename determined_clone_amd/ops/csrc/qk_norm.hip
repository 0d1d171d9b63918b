// RMS norm of queries and keys for each head with the rotary position encoding in the same pass,
// forward and backward, both tensors in one launch.
//
// A head's row x [D] at position p:  r = 1 / sqrt(mean(x^2) + eps),  n = r x,  y = R(p) (w n), where
// R turns the pairs (i, i + rot/2), i < rot/2, by the table's angles and leaves features past rot.
// Backward:  g = R(p)^T dy,  dw = sum over rows of g n,  dx = r (g w - n mean(g w n)).
//
// Bound by HBM: 2 passes forward (x in, y out), 3 backward (x and dy in, dx out). A row takes L lanes
// (the power of two at or above D / V), so a wave works on 64 / L heads of one token at a time and
// walks through its q heads, then its k heads: the angles and the weights stay in registers for the
// whole token. The rotation's partner values come by a second load of the same cache lines, not by
// cross-lane moves: it leaves together with the first one, and the two halves need no alignment to
// lanes. q and k are read through their strides (views of a fused projection).
#include "qk_norm_api.h"

namespace dca {
namespace {

constexpr int kQkWaves = 4;
constexpr int kQkBlock = kQkWaves * 64;

// Sum over each aligned group of L lanes, in every lane of it.
template <int L>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (L >= 2) v += dpp_f32<0xB1>(v);
  if constexpr (L >= 4) v += dpp_f32<0x4E>(v);
  if constexpr (L >= 8) v += dpp_f32<0x141>(v);
  if constexpr (L >= 16) v += dpp_f32<0x140>(v);
  if constexpr (L >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  if constexpr (L >= 64) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  }
  return v;
}

// What a lane keeps for its NV vectors of V features: their columns, the partner columns, the
// weights and, for the current token, the angles (sin with the sign of the partner's term).
template <int V, int NV>
struct Lane {
  int col[NV];    // -1: past D
  int other[NV];  // partner column, -1: not rotated
};

template <typename T, int V, int L, int NV>
__device__ __forceinline__ Lane<V, NV> lane_columns(int D, int rot) {
  Lane<V, NV> a;
  const int l = threadIdx.x & (L - 1), half = rot / 2;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (l + i * L) * V;
    a.col[i] = c < D ? c : -1;
    a.other[i] = c < half ? c + half : (c < rot ? c - half : -1);
  }
  return a;
}

template <int V>
__device__ __forceinline__ void load_f32(const float* p, int64_t at, float (&out)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) out[k] = p[at + k];
}

// Angles of token t: row `at` of the tables, NaN when it has no row there.
template <int V, int NV>
__device__ __forceinline__ void load_angles(const QkShape& s, const float* __restrict__ cosT,
                                            const float* __restrict__ sinT, int64_t b, int64_t tok,
                                            const Lane<V, NV>& a, float sign, float (&cs)[NV][V],
                                            float (&sn)[NV][V]) {
  if (s.rot == 0) return;
  const int64_t at = s.pos.p ? s.pos.at(b * s.pos_sb + tok) : tok;
  const bool ok = static_cast<uint64_t>(at) < static_cast<uint64_t>(s.table_rows);
  const int half = s.rot / 2;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (a.other[i] < 0) continue;
    const bool low = a.other[i] > a.col[i];
    const int64_t c = at * half + (low ? a.col[i] : a.other[i]);
    if (ok) {
      load_f32<V>(cosT, c, cs[i]);
      load_f32<V>(sinT, c, sn[i]);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      cs[i][k] = ok ? cs[i][k] : __builtin_nanf("");
      sn[i][k] = ok ? (low ? -sign : sign) * sn[i][k] : __builtin_nanf("");
    }
  }
}

__device__ __forceinline__ int64_t head_offset(const HeadView& v, int64_t b, int64_t t, int h) {
  return b * v.sb + t * v.ss + h * v.sh;
}

template <typename T, int V, int L, int NV>
__global__ __launch_bounds__(kQkBlock) void qk_fwd_kernel(QkShape s, HeadView xq, HeadView xk, HeadView yq,
                                                          HeadView yk, const float* __restrict__ wq,
                                                          const float* __restrict__ wk,
                                                          const float* __restrict__ cosT,
                                                          const float* __restrict__ sinT) {
  constexpr int G = 64 / L;  // heads at a time
  const Lane<V, NV> a = lane_columns<T, V, L, NV>(s.D, s.rot);
  const int group = (threadIdx.x & 63) / L;
  const int64_t tokens = s.B * s.S, step = static_cast<int64_t>(gridDim.x) * kQkWaves;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kQkWaves + (threadIdx.x >> 6); t < tokens; t += step) {
    const int64_t b = t / s.S, tok = t - b * s.S;
    float cs[NV][V], sn[NV][V];
    load_angles<V, NV>(s, cosT, sinT, b, tok, a, 1.f, cs, sn);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const HeadView& x = which ? xk : xq;
      const HeadView& y = which ? yk : yq;
      const float* __restrict__ w = which ? wk : wq;
      for (int h = group + static_cast<int>(blockIdx.y) * G; h < s.heads[which]; h += G * static_cast<int>(gridDim.y)) {
        const int64_t xo = head_offset(x, b, tok, h), yo = head_offset(y, b, tok, h);
        RawVec<T, V> rx[NV], ro[NV];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (a.col[i] >= 0) rx[i] = ldv<T, V>(x.p, xo + a.col[i]);
          if (a.other[i] >= 0) ro[i] = ldv<T, V>(x.p, xo + a.other[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (a.col[i] < 0) continue;
          float v[V];
          unpackv<T, V>(rx[i], v);
#pragma unroll
          for (int k = 0; k < V; ++k) ss += v[k] * v[k];
        }
        const float r = 1.f / sqrtf(group_sum<L>(ss) / static_cast<float>(s.D) + s.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (a.col[i] < 0) continue;
          float v[V], wv[V];
          unpackv<T, V>(rx[i], v);
          if (w) load_f32<V>(w, a.col[i], wv);
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] *= w ? r * wv[k] : r;
          if (a.other[i] >= 0) {
            float o[V];
            unpackv<T, V>(ro[i], o);
            if (w) load_f32<V>(w, a.other[i], wv);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = v[k] * cs[i][k] + o[k] * (w ? r * wv[k] : r) * sn[i][k];
          }
          stv<T, V>(y.p, yo + a.col[i], packv<T, V>(v));
        }
      }
    }
  }
}

template <typename T, int V, int L, int NV>
__global__ __launch_bounds__(kQkBlock) void qk_bwd_kernel(QkShape s, HeadView gq, HeadView gk, HeadView xq,
                                                          HeadView xk, HeadView dq, HeadView dk,
                                                          const float* __restrict__ wq,
                                                          const float* __restrict__ wk,
                                                          const float* __restrict__ cosT,
                                                          const float* __restrict__ sinT,
                                                          float* __restrict__ partial) {
  constexpr int G = 64 / L;
  __shared__ float red[kQkWaves][L * NV * V];
  const Lane<V, NV> a = lane_columns<T, V, L, NV>(s.D, s.rot);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane / L;
  const int64_t tokens = s.B * s.S, step = static_cast<int64_t>(gridDim.x) * kQkWaves;
  float dw[2][NV][V];
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) dw[which][i][k] = 0.f;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kQkWaves + wave; t < tokens; t += step) {
    const int64_t b = t / s.S, tok = t - b * s.S;
    float cs[NV][V], sn[NV][V];
    load_angles<V, NV>(s, cosT, sinT, b, tok, a, -1.f, cs, sn);  // the transpose turns back
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const HeadView& x = which ? xk : xq;
      const HeadView& y = which ? gk : gq;
      const HeadView& d = which ? dk : dq;
      const float* __restrict__ w = which ? wk : wq;
      for (int h = group + static_cast<int>(blockIdx.y) * G; h < s.heads[which]; h += G * static_cast<int>(gridDim.y)) {
        const int64_t xo = head_offset(x, b, tok, h), yo = head_offset(y, b, tok, h);
        RawVec<T, V> rx[NV], rg[NV], ro[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (a.col[i] >= 0) {
            rx[i] = ldv<T, V>(x.p, xo + a.col[i]);
            rg[i] = ldv<T, V>(y.p, yo + a.col[i]);
          }
          if (a.other[i] >= 0) ro[i] = ldv<T, V>(y.p, yo + a.other[i]);
        }
        float g[NV][V], ss = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (a.col[i] < 0) continue;
          float v[V];
          unpackv<T, V>(rx[i], v);
          unpackv<T, V>(rg[i], g[i]);
          if (a.other[i] >= 0) {
            float o[V];
            unpackv<T, V>(ro[i], o);
#pragma unroll
            for (int k = 0; k < V; ++k) g[i][k] = g[i][k] * cs[i][k] + o[k] * sn[i][k];
          }
          float wv[V];
          if (w) load_f32<V>(w, a.col[i], wv);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            ss += v[k] * v[k];
            dot += (w ? g[i][k] * wv[k] : g[i][k]) * v[k];
          }
        }
        const float r = 1.f / sqrtf(group_sum<L>(ss) / static_cast<float>(s.D) + s.eps);
        const float m = group_sum<L>(dot) / static_cast<float>(s.D) * r * r;  // mean(g w n) r
        const int64_t o = head_offset(d, b, tok, h);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (a.col[i] < 0) continue;
          float v[V], wv[V];
          unpackv<T, V>(rx[i], v);
          if (w) load_f32<V>(w, a.col[i], wv);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            dw[which][i][k] += g[i][k] * (v[k] * r);
            v[k] = r * ((w ? g[i][k] * wv[k] : g[i][k]) - v[k] * m);
          }
          stv<T, V>(d.p, o + a.col[i], packv<T, V>(v));
        }
      }
    }
  }
  if (!partial) return;
  // the workgroup's row of sums: lane groups, then waves, in a fixed order
  const int64_t row = static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float v = dw[which][i][k];
#pragma unroll
        for (int off = 32; off >= L; off >>= 1) v += __shfl_xor(v, off, 64);
        if (group == 0) red[wave][(lane + i * L) * V + k] = v;
      }
    __syncthreads();
    for (int c = threadIdx.x; c < s.D; c += kQkBlock)
      partial[(row * 2 + which) * s.D + c] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
    __syncthreads();
  }
}

// dw[c] (+)= sum of the partial rows of q (columns 0 .. D-1) or k (the rest), 16 waves, fixed order
constexpr int kSumWaves = 16;
__global__ __launch_bounds__(kSumWaves * 64) void qk_dw_kernel(const float* __restrict__ partial, int rows, int D,
                                                               ColumnOut q, ColumnOut k) {
  __shared__ float red[kSumWaves][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float a = 0.f;
  if (c < 2 * D)
#pragma unroll 4
    for (int i = w; i < rows; i += kSumWaves) a += partial[static_cast<int64_t>(i) * 2 * D + c];
  red[w][lane] = a;
  __syncthreads();
  if (w || c >= 2 * D) return;
  for (int i = 1; i < kSumWaves; ++i) a += red[i][lane];
  const ColumnOut& o = c < D ? q : k;
  const int j = c < D ? c : c - D;
  if (!o.p0) return;
  if (o.bf16) {
    uint16_t* p = static_cast<uint16_t*>(o.p0) + j;
    if (o.accumulate) a += __uint_as_float(static_cast<uint32_t>(*p) << 16);
    *p = static_cast<uint16_t>(f2bf_bits(a));
  } else {
    float* p = static_cast<float*>(o.p0) + j;
    *p = o.accumulate ? *p + a : a;
  }
}

// f(T, V, L, NV) for the row length: full vectors keep a row in one vector per lane; narrower ones
// (odd lengths, strides or rotated parts) take the whole wave for a row.
template <typename T, int V, typename F>
void dispatch_lanes(int D, F&& f) {
  const int n = (D + V - 1) / V;
  if constexpr (V == kFull<T>) {
    if (n <= 8) f(T{}, VTag<V>{}, VTag<8>{}, VTag<1>{});
    else if (n <= 16) f(T{}, VTag<V>{}, VTag<16>{}, VTag<1>{});
    else if (n <= 32) f(T{}, VTag<V>{}, VTag<32>{}, VTag<1>{});
    else if (n <= 64) f(T{}, VTag<V>{}, VTag<64>{}, VTag<1>{});
    else if (n <= 128) f(T{}, VTag<V>{}, VTag<64>{}, VTag<2>{});
    else f(T{}, VTag<V>{}, VTag<64>{}, VTag<4>{});
  } else {
    if (n <= 64) f(T{}, VTag<V>{}, VTag<64>{}, VTag<1>{});
    else if (n <= 128) f(T{}, VTag<V>{}, VTag<64>{}, VTag<2>{});
    else if (n <= 256) f(T{}, VTag<V>{}, VTag<64>{}, VTag<4>{});
    else if (n <= 512) f(T{}, VTag<V>{}, VTag<64>{}, VTag<8>{});
    else f(T{}, VTag<V>{}, VTag<64>{}, VTag<16>{});
  }
}
template <typename T, typename F>
void dispatch_row(int vec_bytes, int D, F&& f) {
  dispatch_v<T>(vec_bytes, [&](auto t, auto v) { dispatch_lanes<decltype(t), decltype(v)::value>(D, f); });
}
template <typename F>
void dispatch_all(TDtype dt, int vec_bytes, int D, F&& f) {
  switch (dt) {
    case TDtype::kBF16: dispatch_row<BF16>(vec_bytes, D, f); break;
    case TDtype::kF16: dispatch_row<F16>(vec_bytes, D, f); break;
    default: dispatch_row<F32>(vec_bytes, D, f); break;
  }
}

// Workgroups: a wave a token up to kMaxBlocks of them, and several workgroups a token (over its
// heads) while tokens alone leave the chip empty. `backward` writes a partial row per workgroup.
constexpr int kMaxBlocks = 2048;
dim3 qk_grid(const QkShape& s, int heads_at_once) {
  int64_t x = (s.B * s.S + kQkWaves - 1) / kQkWaves;
  x = x < 1 ? 1 : (x > kMaxBlocks ? kMaxBlocks : x);
  const int most = s.heads[0] > s.heads[1] ? s.heads[0] : s.heads[1];
  int64_t y = (most + heads_at_once - 1) / heads_at_once;
  if (y > 256 / x) y = 256 / x;
  if (y < 1) y = 1;
  return dim3(static_cast<unsigned>(x), static_cast<unsigned>(y));
}
}  // namespace

void qk_norm_rope_fwd(TDtype dt, int vec_bytes, const QkShape& s, const HeadView x[2], const HeadView y[2],
                      const float* const w[2], const float* cosT, const float* sinT, hipStream_t st) {
  if (s.B * s.S == 0 || s.heads[0] + s.heads[1] == 0 || s.D == 0) return;
  dispatch_all(dt, vec_bytes, s.D, [&](auto t, auto v, auto l, auto nv) {
    constexpr int L = decltype(l)::value;
    hipLaunchKernelGGL((qk_fwd_kernel<decltype(t), decltype(v)::value, L, decltype(nv)::value>),
                       qk_grid(s, 64 / L), dim3(kQkBlock), 0, st, s, x[0], x[1], y[0], y[1], w[0], w[1], cosT,
                       sinT);
  });
}

int64_t qk_norm_rope_partial_floats(const QkShape& s) {
  const dim3 g = qk_grid(s, 1);  // at least as many workgroups as any variant launches
  return static_cast<int64_t>(g.x) * g.y * 2 * s.D;
}

void qk_norm_rope_bwd(TDtype dt, int vec_bytes, const QkShape& s, const HeadView dy[2], const HeadView x[2],
                      const HeadView dx[2], const float* const w[2], const float* cosT, const float* sinT,
                      float* partial, const ColumnOut* const dw[2], hipStream_t st) {
  const bool want = dw[0] || dw[1];
  int rows = 0;
  if (s.B * s.S > 0 && s.heads[0] + s.heads[1] > 0 && s.D > 0) {
    dispatch_all(dt, vec_bytes, s.D, [&](auto t, auto v, auto l, auto nv) {
      constexpr int L = decltype(l)::value;
      const dim3 grid = qk_grid(s, 64 / L);
      rows = static_cast<int>(grid.x * grid.y);
      hipLaunchKernelGGL((qk_bwd_kernel<decltype(t), decltype(v)::value, L, decltype(nv)::value>), grid,
                         dim3(kQkBlock), 0, st, s, dy[0], dy[1], x[0], x[1], dx[0], dx[1], w[0], w[1], cosT,
                         sinT, want ? partial : nullptr);
    });
  }
  if (!want || s.D == 0) return;
  hipLaunchKernelGGL(qk_dw_kernel, dim3((2 * s.D + 63) / 64), dim3(kSumWaves * 64), 0, st, partial, rows, s.D,
                     dw[0] ? *dw[0] : ColumnOut{}, dw[1] ? *dw[1] : ColumnOut{});
}
}  // namespace dca
