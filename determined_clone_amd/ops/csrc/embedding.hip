// Token embedding with scaling, learned positions and vocabulary shards, and its gradient.
//
// Forward: out[t] = scale * W[id_t] + P[pos_t] in fp32, rounded once.
//
// Gradient: dW[v] = scale * sum_{t: id_t = v} dy[t]. The ids are sorted (stably, so that a token's
// rows are added in token order and the result does not depend on scheduling), and workgroups take
// equal ranges of the SORTED order: a frequent token is spread over as many workgroups as its rows
// need, a rare one costs one row. A token inside one range is written once; one that crosses ranges
// leaves fp32 partial rows which a second kernel joins in order. No float atomics.
//
// The sort is a least-significant-digit radix sort of chunks in LDS (one workgroup a chunk), and
// merges of up to 16 sorted chunks in which every element finds its rank by binary searches: ids
// are few (16k-64k) beside the rows they index, so what counts is launches and latency.
#include "embedding_api.h"

namespace dca {
namespace {

// ------------------------------------------------------------------ forward
constexpr int kFwdBlock = 256;
constexpr int kFwdUnroll = 4;

template <typename T, int V>
__global__ __launch_bounds__(kFwdBlock) void embed_fwd_kernel(
    EmbedIds ids, const void* __restrict__ table, int64_t stride, EmbedPos pos, float scale,
    void* __restrict__ out, int E, int rows_per_block) {
  const unsigned nv = static_cast<unsigned>(E / V);
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * rows_per_block;
  const int64_t left = ids.n - t0;
  const unsigned n = static_cast<unsigned>(left < rows_per_block ? left : rows_per_block) * nv;
  for (unsigned i0 = threadIdx.x; i0 < n; i0 += kFwdBlock * kFwdUnroll) {
    RawVec<T, V> w[kFwdUnroll], p[kFwdUnroll];
    bool wok[kFwdUnroll], pok[kFwdUnroll];
#pragma unroll
    for (int u = 0; u < kFwdUnroll; ++u) {
      const unsigned i = i0 + u * kFwdBlock;
      wok[u] = pok[u] = false;
      if (i >= n) continue;
      const unsigned r = i / nv;
      const int64_t c = static_cast<int64_t>(i - r * nv) * V, t = t0 + r;
      const int64_t id = ids.ids.at(t) - ids.start;
      wok[u] = static_cast<uint64_t>(id) < static_cast<uint64_t>(ids.rows);
      if (wok[u]) w[u] = ldv<T, V>(table, id * stride + c);
      if (pos.rows) {
        const int64_t at = pos.ids.p ? pos.ids.at(t) : t % pos.S;
        pok[u] = static_cast<uint64_t>(at) < static_cast<uint64_t>(pos.rows);
        if (pok[u]) p[u] = ldv<T, V>(pos.table, at * pos.stride + c);
      }
    }
#pragma unroll
    for (int u = 0; u < kFwdUnroll; ++u) {
      const unsigned i = i0 + u * kFwdBlock;
      if (i >= n) continue;
      float a[V], b[V];
      const float none = ids.shard ? 0.f : __builtin_nanf("");
      if (wok[u]) unpackv<T, V>(w[u], a);
#pragma unroll
      for (int k = 0; k < V; ++k) a[k] = wok[u] ? a[k] * scale : none;
      if (pos.rows) {
        if (pok[u]) unpackv<T, V>(p[u], b);
#pragma unroll
        for (int k = 0; k < V; ++k) a[k] = pok[u] ? a[k] + b[k] : __builtin_nanf("");
      }
      stv<T, V>(out, t0 * E + static_cast<int64_t>(i) * V, packv<T, V>(a));
    }
  }
}

// ------------------------------------------------------------------ sort
// An entry is row << 32 | token index: all entries differ, and their order is the stable one.
constexpr int kSortItems = 4;
constexpr int kSortChunk = 1024 * kSortItems;
constexpr int kDigits = 256;
constexpr int kMergeWays = 16;

__device__ __forceinline__ int row_of(uint64_t entry) { return static_cast<int>(entry >> 32); }

// Sorts one chunk of ids per workgroup by row, least significant digit first. Per digit every wave
// counts its own items in order (lanes with equal digits find each other by ballots), one scan over
// (digit, wave) turns counts into places, and the items move through LDS. Rows past the table
// (other shards, mistakes, the padding of the last chunk) take the key `rows`, after all others.
__global__ __launch_bounds__(1024) void embed_sort_kernel(EmbedIds ids, uint64_t* __restrict__ out, int bits) {
  __shared__ uint64_t buf[kSortChunk];
  __shared__ uint32_t count[16 * kDigits];
  __shared__ uint32_t wave_total[16];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kSortChunk;
  const int n = static_cast<int>(ids.n - base < kSortChunk ? ids.n - base : kSortChunk);
  const uint64_t below = (1ull << lane) - 1;
  volatile uint32_t* mine = count + w * kDigits;  // volatile: a wave's own reads and writes stay in order
  uint32_t key[kSortItems], at[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int l = (w * kSortItems + j) * 64 + lane;
    key[j] = static_cast<uint32_t>(ids.rows);
    at[j] = static_cast<uint32_t>(base + l);
    if (l < n) {
      const int64_t id = ids.ids.at(base + l) - ids.start;
      if (static_cast<uint64_t>(id) < static_cast<uint64_t>(ids.rows)) key[j] = static_cast<uint32_t>(id);
    }
  }
  for (int shift = 0; shift < bits; shift += 8) {
#pragma unroll
    for (int i = 0; i < kDigits / 64; ++i) mine[i * 64 + lane] = 0;
    uint32_t rank[kSortItems];
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
      const uint32_t d = (key[j] >> shift) & (kDigits - 1);
      uint64_t same = ~0ull;
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const bool one = (d >> b) & 1;
        const uint64_t v = __ballot(one);
        same &= one ? v : ~v;
      }
      const uint32_t before = static_cast<uint32_t>(__popcll(same & below));
      const uint32_t had = mine[d];
      rank[j] = had + before;
      if (before == 0) mine[d] = had + static_cast<uint32_t>(__popcll(same));
    }
    __syncthreads();
    // exclusive scan over (digit, wave): thread t takes digit t / 4, waves 4 (t % 4) .. + 3
    const int sd = tid >> 2, sw = (tid & 3) * 4;
    uint32_t c[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = count[(sw + i) * kDigits + sd];
      sum += c[i];
    }
    uint32_t incl = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint32_t v = __shfl_up(incl, off, 64);
      if (lane >= off) incl += v;
    }
    if (lane == 63) wave_total[w] = incl;
    __syncthreads();
    uint32_t place = incl - sum;
    for (int i = 0; i < w; ++i) place += wave_total[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      count[(sw + i) * kDigits + sd] = place;
      place += c[i];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortItems; ++j)
      buf[count[w * kDigits + ((key[j] >> shift) & (kDigits - 1))] + rank[j]] =
          static_cast<uint64_t>(key[j]) << 32 | at[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
      const uint64_t e = buf[(w * kSortItems + j) * 64 + lane];
      key[j] = static_cast<uint32_t>(e >> 32);
      at[j] = static_cast<uint32_t>(e);
    }
  }
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int l = (w * kSortItems + j) * 64 + lane;
    if (l < n) out[base + l] = static_cast<uint64_t>(key[j]) << 32 | at[j];
  }
}

// Merges groups of up to kMergeWays sorted runs of `len`: an element's place is its own index plus
// the number of smaller elements in each of the group's other runs.
__global__ __launch_bounds__(256) void embed_merge_kernel(const uint64_t* __restrict__ in,
                                                          uint64_t* __restrict__ out, int64_t n,
                                                          int64_t len) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  const uint64_t v = in[i];
  const int64_t run = i / len;
  const int64_t g0 = run / kMergeWays * kMergeWays;  // the group's first run
  int64_t place = g0 * len + (i - run * len);
  int64_t top = 1;
  while (top * 2 <= len) top *= 2;
#pragma unroll 4
  for (int k = 0; k < kMergeWays; ++k) {
    const int64_t r0 = (g0 + k) * len;
    const int64_t m = n - r0 < len ? n - r0 : len;
    if (m <= 0 || g0 + k == run) continue;
    int64_t below = 0;
    for (int64_t step = top; step > 0; step >>= 1)
      if (below + step <= m && in[r0 + below + step - 1] < v) below += step;
    place += below;
  }
  out[place] = v;
}

// ------------------------------------------------------------------ gradient
constexpr int kGradUnroll = 8;

__device__ __forceinline__ int64_t partial_stride(int E) { return (E + 3) & ~3; }

template <typename T, int V>
__device__ __forceinline__ void grad_store(void* out, int64_t at, float (&a)[V], float scale, bool accumulate) {
#pragma unroll
  for (int k = 0; k < V; ++k) a[k] *= scale;
  if (accumulate) {
    float old[V];
    unpackv<T, V>(ldv<T, V>(out, at), old);
#pragma unroll
    for (int k = 0; k < V; ++k) a[k] += old[k];
  }
  stv<T, V>(out, at, packv<T, V>(a));
}

// Workgroup x takes sorted entries [x K, (x + 1) K), workgroup y a stretch of columns. partial
// holds two rows a workgroup: 0 the sum of a token that began in an earlier range (its "head"),
// 1 of one that began here and goes on (its "tail").
template <typename T, int V>
__global__ __launch_bounds__(256) void embed_grad_kernel(const uint64_t* __restrict__ sorted,
                                                         const void* __restrict__ dy, void* __restrict__ out,
                                                         float* __restrict__ partial, int64_t n, int64_t rows,
                                                         int E, int K, float scale, bool accumulate) {
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  const bool ok = c < E;
  const int64_t lo = static_cast<int64_t>(blockIdx.x) * K;
  const int64_t hi = lo + K < n ? lo + K : n;
  const int64_t ps = partial_stride(E);
  float* head = partial + static_cast<int64_t>(blockIdx.x) * 2 * ps;
  int row = row_of(sorted[lo]);
  bool open = lo > 0 && row_of(sorted[lo - 1]) == row;
  float a[V];
#pragma unroll
  for (int k = 0; k < V; ++k) a[k] = 0.f;
  auto put = [&](float* to) {
    if (!ok) return;
#pragma unroll
    for (int k = 0; k < V; ++k) to[c + k] = a[k];
  };
  for (int64_t e = lo; e < hi; e += kGradUnroll) {
    if (row_of(sorted[e]) >= rows) break;  // rows of no table: all that follow are, too
    uint64_t s[kGradUnroll];
    RawVec<T, V> r[kGradUnroll];
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u) s[u] = sorted[e + u < hi ? e + u : hi - 1];
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u)
      if (ok) r[u] = ldv<T, V>(dy, static_cast<int64_t>(s[u] & 0xffffffffu) * E + c);
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u) {
      if (e + u >= hi) continue;
      const int next = row_of(s[u]);
      if (next != row) {
        if (open) put(head);
        else if (ok && row < rows) grad_store<T, V>(out, static_cast<int64_t>(row) * E + c, a, scale, accumulate);
#pragma unroll
        for (int k = 0; k < V; ++k) a[k] = 0.f;
        row = next;
        open = false;
      }
      if (ok) {
        float x[V];
        unpackv<T, V>(r[u], x);
#pragma unroll
        for (int k = 0; k < V; ++k) a[k] += x[k];
      }
    }
  }
  if (row >= rows) return;
  if (open) put(head);
  else if (hi < n && row_of(sorted[hi]) == row) put(head + ps);
  else if (ok) grad_store<T, V>(out, static_cast<int64_t>(row) * E + c, a, scale, accumulate);
}

// Joins the tokens that cross ranges: the workgroup in whose range a token begins adds the heads of
// the following ranges to its tail. 4 waves take every fourth range, 256 columns a workgroup.
constexpr int kJoinWaves = 4;
template <typename T>
__global__ __launch_bounds__(kJoinWaves * 64) void embed_join_kernel(const uint64_t* __restrict__ sorted,
                                                                     const float* __restrict__ partial,
                                                                     void* __restrict__ out, int64_t n,
                                                                     int64_t rows, int E, int K, float scale,
                                                                     bool accumulate) {
  __shared__ float4 red[kJoinWaves][64];
  const int64_t lo = static_cast<int64_t>(blockIdx.x) * K, hi = lo + K;
  if (hi >= n) return;
  const int row = row_of(sorted[hi - 1]);
  if (row >= rows || row_of(sorted[hi]) != row) return;                                  // ends here
  if (lo > 0 && row_of(sorted[lo]) == row && row_of(sorted[lo - 1]) == row) return;      // began earlier
  // the last range that holds the token: doubling steps, then halving ones
  const int64_t x = blockIdx.x, nb = (n + K - 1) / K;
  int64_t last = x + 1, step = 1;  // range `last` begins with the token
  while (last + step < nb && row_of(sorted[(last + step) * K]) == row) {
    last += step;
    step *= 2;
  }
  for (; step > 0; step >>= 1)
    if (last + step < nb && row_of(sorted[(last + step) * K]) == row) last += step;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = (blockIdx.y * 64 + lane) * 4;
  const int64_t ps = partial_stride(E);
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < E) {
#pragma unroll 4
    for (int64_t b = x + 1 + w; b <= last; b += kJoinWaves) {
      const float4 p = *reinterpret_cast<const float4*>(partial + b * 2 * ps + c);
      a.x += p.x; a.y += p.y; a.z += p.z; a.w += p.w;
    }
  }
  red[w][lane] = a;
  __syncthreads();
  if (w || c >= E) return;
  a = *reinterpret_cast<const float4*>(partial + (x * 2 + 1) * ps + c);
#pragma unroll
  for (int i = 0; i < kJoinWaves; ++i) {
    const float4 p = red[i][lane];
    a.x += p.x; a.y += p.y; a.z += p.z; a.w += p.w;
  }
  const float v[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (c + k >= E) break;
    float one[1] = {v[k]};
    grad_store<T, 1>(out, static_cast<int64_t>(row) * E + c + k, one, scale, accumulate);
  }
}

// ------------------------------------------------------------------ position gradient
// Column sums of dy [B][N]: a lane takes V columns, the workgroup's waves split the batch and join
// in a fixed order.
constexpr int kSumUnroll = 8;
template <typename T, int V>
__global__ __launch_bounds__(1024) void batch_sum_kernel(const void* __restrict__ dy, void* __restrict__ out,
                                                         int64_t B, int64_t N, bool accumulate) {
  extern __shared__ float red[];  // [waves][64][V]
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * 64 + lane) * V;
  float a[V];
#pragma unroll
  for (int k = 0; k < V; ++k) a[k] = 0.f;
  if (c < N) {
    for (int64_t b = w; b < B; b += static_cast<int64_t>(waves) * kSumUnroll) {
      RawVec<T, V> r[kSumUnroll];
#pragma unroll
      for (int u = 0; u < kSumUnroll; ++u)
        if (b + u * waves < B) r[u] = ldv<T, V>(dy, (b + u * waves) * N + c);
#pragma unroll
      for (int u = 0; u < kSumUnroll; ++u) {
        if (b + u * waves >= B) continue;
        float x[V];
        unpackv<T, V>(r[u], x);
#pragma unroll
        for (int k = 0; k < V; ++k) a[k] += x[k];
      }
    }
  }
  if (waves > 1) {
#pragma unroll
    for (int k = 0; k < V; ++k) red[(w * 64 + lane) * V + k] = a[k];
    __syncthreads();
    if (w) return;
    for (int i = 1; i < waves; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) a[k] += red[(i * 64 + lane) * V + k];
  }
  if (c < N) grad_store<T, V>(out, c, a, 1.f, accumulate);
}

template <typename F>
void dispatch_tv(TDtype dt, int vec_bytes, F&& f) {
  switch (dt) {
    case TDtype::kBF16: dispatch_v<BF16>(vec_bytes, f); break;
    case TDtype::kF16: dispatch_v<F16>(vec_bytes, f); break;
    default: dispatch_v<F32>(vec_bytes, f); break;
  }
}

// Sorted entries a workgroup takes: enough workgroups to fill the chip, few partial rows.
int grad_range(int64_t n) { return n >= 16384 ? 32 : (n >= 4096 ? 16 : 8); }

int64_t partial_floats(int64_t n, int E) {
  const int64_t K = grad_range(n);
  return (n + K - 1) / K * 2 * ((E + 3) & ~3);
}
}  // namespace

void embed_fwd(TDtype dt, int vec_bytes, const EmbedIds& ids, const void* table, int64_t stride,
               const EmbedPos& pos, float scale, void* out, int E, hipStream_t st) {
  if (ids.n == 0 || E == 0) return;
  dispatch_tv(dt, vec_bytes, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    const int64_t nv = E / V;
    // one pass of the workgroup's unrolled loop, as long as that leaves 1024 workgroups
    int64_t r = kFwdBlock * kFwdUnroll / nv;
    if (r > ids.n / 1024) r = ids.n / 1024;
    if (r < 1) r = 1;
    hipLaunchKernelGGL((embed_fwd_kernel<T, V>), dim3(static_cast<unsigned>((ids.n + r - 1) / r)),
                       dim3(kFwdBlock), 0, st, ids, table, stride, pos, scale, out, E, static_cast<int>(r));
  });
}

int64_t embed_grad_workspace(int64_t n, int E) { return 2 * n * 8 + partial_floats(n, E) * 4 + 16; }

void embed_grad(TDtype dt, int vec_bytes, const EmbedIds& ids, const void* dy, void* out, int E,
                float scale, bool accumulate, void* workspace, hipStream_t st) {
  const int64_t n = ids.n;
  if (n == 0 || E == 0) return;
  uint64_t* a = static_cast<uint64_t*>(workspace);
  uint64_t* b = a + n;
  float* partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + (2 * n * 8 + 15) / 16 * 16);
  int bits = 1;  // of the largest key, `rows` itself
  while (bits < 32 && (ids.rows >> bits)) ++bits;
  hipLaunchKernelGGL(embed_sort_kernel, dim3(static_cast<unsigned>((n + kSortChunk - 1) / kSortChunk)),
                     dim3(1024), 0, st, ids, a, bits);
  for (int64_t len = kSortChunk; len < n; len *= kMergeWays) {
    hipLaunchKernelGGL(embed_merge_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, st,
                       a, b, n, len);
    uint64_t* t = a;
    a = b;
    b = t;
  }
  const int K = grad_range(n);
  const unsigned nb = static_cast<unsigned>((n + K - 1) / K);
  dispatch_tv(dt, vec_bytes, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    const int nv = E / V;
    const int threads = nv >= 256 ? 256 : (nv + 63) / 64 * 64;
    hipLaunchKernelGGL((embed_grad_kernel<T, V>), dim3(nb, static_cast<unsigned>((nv + threads - 1) / threads)),
                       dim3(threads), 0, st, a, dy, out, partial, n, ids.rows, E, K, scale, accumulate);
    if (nb > 1)
      hipLaunchKernelGGL(embed_join_kernel<T>, dim3(nb, static_cast<unsigned>((E + 255) / 256)),
                         dim3(kJoinWaves * 64), 0, st, a, partial, out, n, ids.rows, E, K, scale, accumulate);
  });
}

void batch_sum(TDtype dt, int vec_bytes, const void* dy, void* out, int64_t B, int64_t N,
               bool accumulate, hipStream_t st) {
  if (N == 0) return;
  dispatch_tv(dt, vec_bytes, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    const int64_t tiles = (N / V + 63) / 64;
    int waves = 1;  // split the batch where the columns alone do not fill the chip
    while (waves < 16 && waves * 2 <= B && tiles * waves < 4096) waves *= 2;
    hipLaunchKernelGGL((batch_sum_kernel<T, V>), dim3(static_cast<unsigned>(tiles)), dim3(waves * 64),
                       waves > 1 ? static_cast<size_t>(waves) * 64 * V * sizeof(float) : 0, st, dy, out, B, N,
                       accumulate);
  });
}
}  // namespace dca
