// RMS norm of queries and keys for each head with the rotary position encoding in the same pass,
// forward and backward, both tensors in one launch.
//
// A head's row x [D] at position p:  r = 1 / sqrt(mean(x^2) + eps),  n = r x,  y = R(p) (w n), where
// R turns the pairs (i, i + rot/2), i < rot/2, by the table's angles and leaves features past rot.
// Backward:  g = R(p)^T dy,  dw = sum over rows of g n,  dx = r (g w - n mean(g w n)).
//
// Bound by HBM: 2 passes forward (x in, y out), 3 backward (x and dy in, dx out). At 32x1024 tokens,
// 20 + 20 heads of 64 in bf16 (168 MB a pass): forward 73 us, 4.6 TB/s; backward 102 us, 4.9 TB/s; a
// large copy reaches 5.1 TB/s. A row takes L lanes
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

// The columns of a lane's NV vectors of V features.
template <int V, int NV>
struct Lane {
  int col[NV];    // -1: past D
  int other[NV];  // the rotation's partner column, -1: not rotated
};

template <int V, int L, int NV>
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

// Angles of a token: y = x cs + x[partner] sn, with sn's sign for this half of the pair (`sign` -1
// turns back). Features that do not turn have cs 1, sn 0; a position without a table row gives NaN.
template <int V, int NV>
__device__ __forceinline__ void load_angles(const QkShape& s, const float* __restrict__ cosT,
                                            const float* __restrict__ sinT, int64_t b, int64_t tok,
                                            const Lane<V, NV>& a, float sign, float (&cs)[NV][V],
                                            float (&sn)[NV][V]) {
  int64_t at = 0;
  bool ok = true;
  if (s.rot) {
    at = s.pos.p ? s.pos.at(b * s.pos_sb + tok) : tok;
    ok = static_cast<uint64_t>(at) < static_cast<uint64_t>(s.table_rows);
  }
  const int half = s.rot / 2;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      cs[i][k] = 1.f;
      sn[i][k] = 0.f;
    }
    if (a.other[i] < 0) continue;
    const bool low = a.other[i] > a.col[i];
    const int64_t c = at * half + (low ? a.col[i] : a.other[i]);
    if (ok) {
      load_f32<V>(cosT, c, cs[i]);
      load_f32<V>(sinT, c, sn[i]);
    }
    const float f = ok ? (low ? -sign : sign) : __builtin_nanf("");
#pragma unroll
    for (int k = 0; k < V; ++k) {
      sn[i][k] *= f;
      if (!ok) cs[i][k] = f;
    }
  }
}

// 1 / sqrt(mean + eps): v_rsq_f32 is within 1 ulp, below the rounding of the sum that it takes. It
// takes subnormal numbers (tiny rows without an eps) for 0: those are raised by 2^64 before it.
__device__ __forceinline__ float rms_inv(float sum, float inv_d, float eps) {
  const float m = sum * inv_d + eps;
  const bool tiny = m < 0x1p-126f;
  const float r = __builtin_amdgcn_rsqf(tiny ? m * 0x1p64f : m);
  return tiny ? r * 0x1p32f : r;
}

// U groups of heads at once: their loads leave together, before the first is used.
template <typename T, int V, int L, int NV, int U>
__global__ __launch_bounds__(kQkBlock) void qk_fwd_kernel(QkShape s, HeadView xq, HeadView xk, HeadView yq,
                                                          HeadView yk, const float* __restrict__ wq,
                                                          const float* __restrict__ wk,
                                                          const float* __restrict__ cosT,
                                                          const float* __restrict__ sinT) {
  constexpr int G = 64 / L;  // heads at a time
  const Lane<V, NV> a = lane_columns<V, L, NV>(s.D, s.rot);
  const int group = (threadIdx.x & 63) / L;
  const float inv_d = 1.f / static_cast<float>(s.D);
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
      const int heads = s.heads[which];
      // the weights go into the angles: y = r (x (w cs) + x[partner] (w[partner] sn))
      float cw[NV][V], sw[NV][V];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float wv[V], wo[V];
#pragma unroll
        for (int k = 0; k < V; ++k) wv[k] = wo[k] = 1.f;
        if (w && a.col[i] >= 0) load_f32<V>(w, a.col[i], wv);
        if (w && a.other[i] >= 0) load_f32<V>(w, a.other[i], wo);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          cw[i][k] = wv[k] * cs[i][k];
          sw[i][k] = wo[k] * sn[i][k];
        }
      }
      const int64_t x0 = b * x.sb + tok * x.ss, y0 = b * y.sb + tok * y.ss;
      for (int h0 = group + static_cast<int>(blockIdx.y) * G * U; h0 < heads; h0 += G * U * static_cast<int>(gridDim.y)) {
        RawVec<T, V> rx[U][NV], ro[U][NV];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * G;
          const int64_t xo = x0 + h * x.sh;
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            rx[u][i] = ro[u][i] = RawVec<T, V>{};
            if (h < heads && a.col[i] >= 0) rx[u][i] = ldv<T, V>(x.p, xo + a.col[i]);
            if (h < heads && a.other[i] >= 0) ro[u][i] = ldv<T, V>(x.p, xo + a.other[i]);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * G;
          if (h >= heads) break;
          float v[NV][V], ss = 0.f;
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            float o[V];
            unpackv<T, V>(rx[u][i], v[i]);
            unpackv<T, V>(ro[u][i], o);
#pragma unroll
            for (int k = 0; k < V; ++k) {
              ss += v[i][k] * v[i][k];
              v[i][k] = v[i][k] * cw[i][k] + o[k] * sw[i][k];
            }
          }
          const float r = rms_inv(group_sum<L>(ss), inv_d, s.eps);
          const int64_t yo = y0 + h * y.sh;
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            if (a.col[i] < 0) continue;
#pragma unroll
            for (int k = 0; k < V; ++k) v[i][k] *= r;
            stv<T, V>(y.p, yo + a.col[i], packv<T, V>(v[i]));
          }
        }
      }
    }
  }
}

// One group of heads at a time: two at once measured 128 us against 102 us (32x1024 tokens, 20 + 20
// heads of 64, bf16), since their registers leave 3 waves on a SIMD instead of 4.
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
  const Lane<V, NV> a = lane_columns<V, L, NV>(s.D, s.rot);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane / L;
  const float inv_d = 1.f / static_cast<float>(s.D);
  const int64_t tokens = s.B * s.S, step = static_cast<int64_t>(gridDim.x) * kQkWaves;
  float dw[2][NV][V], wv[2][NV][V];
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        dw[which][i][k] = 0.f;
        wv[which][i][k] = 1.f;
      }
      const float* __restrict__ w = which ? wk : wq;
      if (w && a.col[i] >= 0) load_f32<V>(w, a.col[i], wv[which][i]);
    }
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kQkWaves + wave; t < tokens; t += step) {
    const int64_t b = t / s.S, tok = t - b * s.S;
    float cs[NV][V], sn[NV][V];
    load_angles<V, NV>(s, cosT, sinT, b, tok, a, -1.f, cs, sn);  // the transpose turns back
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const HeadView& x = which ? xk : xq;
      const HeadView& y = which ? gk : gq;
      const HeadView& d = which ? dk : dq;
      const int heads = s.heads[which];
      const int64_t x0 = b * x.sb + tok * x.ss, y0 = b * y.sb + tok * y.ss, d0 = b * d.sb + tok * d.ss;
      for (int h = group + static_cast<int>(blockIdx.y) * G; h < heads; h += G * static_cast<int>(gridDim.y)) {
        const int64_t xo = x0 + h * x.sh, yo = y0 + h * y.sh, at = d0 + h * d.sh;
        RawVec<T, V> rx[NV], rg[NV], ro[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          rx[i] = rg[i] = ro[i] = RawVec<T, V>{};
          if (a.col[i] >= 0) {
            rg[i] = ldv<T, V>(y.p, yo + a.col[i]);
            rx[i] = ldv<T, V>(x.p, xo + a.col[i]);
          }
          if (a.other[i] >= 0) ro[i] = ldv<T, V>(y.p, yo + a.other[i]);
        }
        float g[NV][V], v[NV][V], ss = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float o[V];
          unpackv<T, V>(rx[i], v[i]);
          unpackv<T, V>(rg[i], g[i]);
          unpackv<T, V>(ro[i], o);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            g[i][k] = g[i][k] * cs[i][k] + o[k] * sn[i][k];
            ss += v[i][k] * v[i][k];
            dot += g[i][k] * wv[which][i][k] * v[i][k];
          }
        }
        const float r = rms_inv(group_sum<L>(ss), inv_d, s.eps);
        const float m = group_sum<L>(dot) * inv_d * r * r;  // mean(g w n) r
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (a.col[i] < 0) continue;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            dw[which][i][k] += g[i][k] * (v[i][k] * r);
            v[i][k] = r * (g[i][k] * wv[which][i][k] - v[i][k] * m);
          }
          stv<T, V>(d.p, at + a.col[i], packv<T, V>(v[i]));
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

// dw[c] (+)= sum of the partial rows of q (columns 0 .. D-1) or k (the rest): 16 columns a workgroup,
// its 64 lane groups of 16 take every 64th row, in a fixed order.
constexpr int kSumCols = 16;
__global__ __launch_bounds__(1024) void qk_dw_kernel(const float* __restrict__ partial, int rows, int D,
                                                     ColumnOut q, ColumnOut k) {
  constexpr int kSlices = 1024 / kSumCols;
  __shared__ float red[kSlices][kSumCols];
  const int slice = threadIdx.x / kSumCols, col = threadIdx.x % kSumCols, c = blockIdx.x * kSumCols + col;
  float a = 0.f;
  if (c < 2 * D) {
#pragma unroll 8
    for (int i = slice; i < rows; i += kSlices) a += partial[static_cast<int64_t>(i) * 2 * D + c];
  }
  red[slice][col] = a;
  __syncthreads();
  for (int n = kSlices / 2; n > 0; n >>= 1) {
    if (slice < n) red[slice][col] += red[slice + n][col];
    __syncthreads();
  }
  if (slice || c >= 2 * D) return;
  a = red[0][col];
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

// Groups of heads at once in the forward: rows that take one vector per lane have registers for
// several (4 against 2: 72 against 78 us at 32x1024 tokens, 20 + 20 heads of 64, bf16).
constexpr int unroll_of(int L, int NV) { return NV > 1 ? 1 : (L > 16 ? 2 : 4); }

// Workgroups: a wave a token up to `most` of them, and several workgroups a token (over its heads)
// while tokens alone leave the chip empty. The backward writes a partial row per workgroup.
// More of them do not pay: 2048 backward workgroups 102 us, their longer sum 5.9 against 4.6 us.
constexpr int kFwdBlocks = 8192, kBwdBlocks = 1024;
dim3 qk_grid(const QkShape& s, int heads_at_once, int most) {
  int64_t x = (s.B * s.S + kQkWaves - 1) / kQkWaves;
  x = x < 1 ? 1 : (x > most ? most : x);
  const int heads = s.heads[0] > s.heads[1] ? s.heads[0] : s.heads[1];
  int64_t y = (heads + heads_at_once - 1) / heads_at_once;
  if (y > 256 / x) y = 256 / x;
  if (y < 1) y = 1;
  return dim3(static_cast<unsigned>(x), static_cast<unsigned>(y));
}
}  // namespace

void qk_norm_rope_fwd(TDtype dt, int vec_bytes, const QkShape& s, const HeadView x[2], const HeadView y[2],
                      const float* const w[2], const float* cosT, const float* sinT, hipStream_t st) {
  if (s.B * s.S == 0 || s.heads[0] + s.heads[1] == 0 || s.D == 0) return;
  dispatch_all(dt, vec_bytes, s.D, [&](auto t, auto v, auto l, auto nv) {
    constexpr int L = decltype(l)::value, NV = decltype(nv)::value, U = unroll_of(L, NV);
    hipLaunchKernelGGL((qk_fwd_kernel<decltype(t), decltype(v)::value, L, NV, U>),
                       qk_grid(s, 64 / L * U, kFwdBlocks), dim3(kQkBlock), 0, st, s, x[0], x[1], y[0], y[1], w[0], w[1], cosT,
                       sinT);
  });
}

int64_t qk_norm_rope_partial_floats(const QkShape& s) {
  const dim3 g = qk_grid(s, 1, kBwdBlocks);  // at least as many workgroups as any variant launches
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
      const dim3 grid = qk_grid(s, 64 / L, kBwdBlocks);
      rows = static_cast<int>(grid.x * grid.y);
      hipLaunchKernelGGL((qk_bwd_kernel<decltype(t), decltype(v)::value, L, decltype(nv)::value>), grid,
                         dim3(kQkBlock), 0, st, s, dy[0], dy[1], x[0], x[1], dx[0], dx[1], w[0], w[1], cosT,
                         sinT, want ? partial : nullptr);
    });
  }
  if (!want || s.D == 0) return;
  auto sum = [&](const ColumnOut& q, const ColumnOut& k) {
    hipLaunchKernelGGL(qk_dw_kernel, dim3((2 * s.D + kSumCols - 1) / kSumCols), dim3(1024), 0, st, partial, rows, s.D, q,
                       k);
  };
  const ColumnOut q = dw[0] ? *dw[0] : ColumnOut{}, k = dw[1] ? *dw[1] : ColumnOut{};
  if (q.p0 && q.p0 == k.p0) {  // one weight for both, added to its gradient: one after the other
    sum(q, ColumnOut{});
    sum(ColumnOut{}, k);
  } else {
    sum(q, k);
  }
}
}  // namespace dca
