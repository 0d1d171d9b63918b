// Token embedding with scaling, learned positions and vocabulary shards, and its gradient.
//
// Forward: out[t] = scale * W[id_t] + P[pos_t] in fp32, rounded once.
//
// Gradient: dW[v] = scale * sum_{t: id_t = v} dy[t], without float atomics, so that the result does
// not depend on scheduling. With few ids (direct()) a wave per table row looks through all of them and
// adds the rows of those that are its own, in order. More ids are sorted by row (stably), and workgroups
// take equal ranges of the SORTED order: a frequent token is spread over as many workgroups as its
// rows need, a rare one costs one row. A token inside one range is written once; one that crosses
// ranges leaves fp32 partial rows which a second kernel joins in order.
//
// The sort is one launch: workgroup b owns the rows whose low bits are b (256 workgroups, so that
// frequent tokens, which have low ids in most vocabularies, fall to different ones), reads ALL ids,
// counts those of lower workgroups (its place in the result) and its own by row and wave, and writes
// its own out in order. Reading the ids once per workgroup (256 kB from L2 at 32k ids) costs less than
// the passes and the launches of a sort that moves them.
#include "embedding_api.h"

namespace dca {
namespace {

// ------------------------------------------------------------------ forward
constexpr int kFwdBlock = 256;
constexpr int kFwdUnroll = 4;
// Outputs past the L2s are streamed (203 MB: 57 against 66 us), smaller ones stay for their reader.
constexpr int64_t kStreamBytes = 32 << 20;

// Several entries of an index array: their loads leave together.
template <int N>
__device__ __forceinline__ void read_index(const Index& a, int64_t first, const unsigned (&r)[N], int64_t (&out)[N]) {
  if (a.is32) {
#pragma unroll
    for (int u = 0; u < N; ++u) out[u] = static_cast<const int32_t*>(a.p)[first + r[u]];
  } else {
#pragma unroll
    for (int u = 0; u < N; ++u) out[u] = static_cast<const int64_t*>(a.p)[first + r[u]];
  }
}

// A workgroup takes a few rows, vector after vector. All ids of an unrolled step are read, then all
// rows, with mistakes and the end of the stretch replaced by rows that exist: no load waits for
// another of its kind.
template <typename T, bool kAligned, bool kStream>
__global__ __launch_bounds__(kFwdBlock) void embed_fwd_kernel(
    EmbedIds ids, const void* __restrict__ table, int64_t stride, EmbedPos pos, float scale,
    void* __restrict__ out, int E, int rows_per_block) {
  constexpr int V = kFull<T>;
  const unsigned nv = static_cast<unsigned>((E + V - 1) / V);
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * rows_per_block;
  const int64_t left = ids.n - t0;
  const unsigned n = static_cast<unsigned>(left < rows_per_block ? left : rows_per_block) * nv;
  for (unsigned i0 = threadIdx.x; i0 < n; i0 += kFwdBlock * kFwdUnroll) {
    unsigned r[kFwdUnroll], c[kFwdUnroll];
    int64_t id[kFwdUnroll], at[kFwdUnroll];
    uint4 w[kFwdUnroll], p[kFwdUnroll];
#pragma unroll
    for (int u = 0; u < kFwdUnroll; ++u) {
      const unsigned i = i0 + u * kFwdBlock < n ? i0 + u * kFwdBlock : n - 1;
      r[u] = i / nv;
      c[u] = (i - r[u] * nv) * V;
    }
    read_index(ids.ids, t0, r, id);
    if (pos.rows) {
      if (pos.ids.p) {
        read_index(pos.ids, t0, r, at);
      } else {
#pragma unroll
        for (int u = 0; u < kFwdUnroll; ++u)
          at[u] = static_cast<uint32_t>(t0 + r[u]) % static_cast<uint32_t>(pos.S);
      }
    }
#pragma unroll
    for (int u = 0; u < kFwdUnroll; ++u) {
      id[u] -= ids.start;
      if (static_cast<uint64_t>(id[u]) >= static_cast<uint64_t>(ids.rows)) id[u] = -1;
      w[u] = load_row<T, kAligned, false>(table, (id[u] < 0 ? 0 : id[u]) * stride + c[u], E - c[u]);
    }
    if (pos.rows) {
#pragma unroll
      for (int u = 0; u < kFwdUnroll; ++u) {
        if (static_cast<uint64_t>(at[u]) >= static_cast<uint64_t>(pos.rows)) at[u] = -1;
        p[u] = load_row<T, kAligned, false>(pos.table, (at[u] < 0 ? 0 : at[u]) * pos.stride + c[u], E - c[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kFwdUnroll; ++u) {
      if (i0 + u * kFwdBlock >= n) break;
      float a[V], b[V];
      unpackv<T, V>(w[u], a);
      const float none = ids.shard ? 0.f : __builtin_nanf("");
#pragma unroll
      for (int k = 0; k < V; ++k) a[k] = id[u] < 0 ? none : a[k] * scale;
      if (pos.rows) {
        unpackv<T, V>(p[u], b);
#pragma unroll
        for (int k = 0; k < V; ++k) a[k] = at[u] < 0 ? __builtin_nanf("") : a[k] + b[k];
      }
      store_row<T, kAligned, kStream>(out, (t0 + r[u]) * E + c[u], E - c[u], packv<T, V>(a));
    }
  }
}

// ------------------------------------------------------------------ sort
// An entry is row << 32 | token index; ids without a row (another shard's, mistakes) have row -1.
__device__ __forceinline__ int row_of(uint64_t entry) { return static_cast<int>(entry >> 32); }

constexpr int kPlaceUnroll = 8;
constexpr int kList = 256;
constexpr int kCrowd = 8;

// 16 bytes of zeros at a time, the last bytes one by one; `p` is 16-byte aligned. Not streamed: that
// measured 34 against 28 us beside the sort (161 MB).
__device__ __forceinline__ void zero_fill(void* p, int64_t bytes, int64_t first, int64_t step) {
  const int64_t n = bytes / 16;
  for (int64_t i = first; i < n; i += step) store_row<F32, true, false>(p, i * 4, 4, make_uint4(0, 0, 0, 0));
  if (first < bytes % 16) static_cast<char*>(p)[n * 16 + first] = 0;
}

// A wave's own LDS accesses are carried out in the order they are issued: the compiler keeps it.
__device__ __forceinline__ void keep_order() { asm volatile("" ::: "memory"); }

// Workgroups [0, 2^shift): the sort; b owns the ids with b in their low bits, rows r with r mod 2^shift
// = b and, behind them, the ids that have no row (counter kRows - 1). The others clear `clear`
// meanwhile. A wave walks through its stretch of the ids, 64 at a time, counts, and lists its own in
// LDS; after the scan it places those (with more than kList of them, by walking through its stretch
// again). What bounds it is the instructions per id of the walk, which therefore looks at low bits
// only: whether an id has a row is asked of the few that are the workgroup's own. 32k ids: 4.5 us for
// the walk, beside 4 us of launch, scan and ends.
template <typename I, int kRows, int kWaves>
__global__ __launch_bounds__(kWaves * 64) void embed_place_kernel(const I* __restrict__ ids, int64_t n, int64_t start,
                                                                  int64_t rows, int shift,
                                                                  uint64_t* __restrict__ sorted,
                                                                  void* __restrict__ clear, int64_t clear_bytes) {
  constexpr int kThreads = kWaves * 64, kEach = kRows * kWaves / kThreads;
  const uint32_t owners = 1u << shift;
  if (blockIdx.x >= owners) {
    zero_fill(clear, clear_bytes, static_cast<int64_t>(blockIdx.x - owners) * kThreads + threadIdx.x,
              static_cast<int64_t>(gridDim.x - owners) * kThreads);
    return;
  }
  __shared__ uint32_t count[kWaves * kRows];
  __shared__ uint32_t wave_sum[2][kWaves];
  __shared__ uint32_t list[kWaves][kList];  // counter << 22 | index in the wave's stretch
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t me = blockIdx.x, mask = owners - 1, start_lo = static_cast<uint32_t>(start);
  auto counter_of = [&](I id) {
    const int64_t row = static_cast<int64_t>(id) - start;
    return static_cast<uint64_t>(row) < static_cast<uint64_t>(rows) ? static_cast<uint32_t>(row) >> shift : kRows - 1u;
  };
  // of the lanes in `own`, those with this lane's counter: one counter at a time, and bit by bit where
  // there are many
  auto peers = [&](uint64_t own, uint32_t d) {
    uint64_t left = own, same = 0;
    const bool in = own >> lane & 1;
    for (int k = 0; k < 3 && left; ++k) {
      const uint32_t one = __builtin_amdgcn_readlane(d, __builtin_ctzll(left));
      const uint64_t s = __builtin_amdgcn_ballot_w64(in && d == one);
      if (s >> lane & 1) same = s;
      left &= ~s;
    }
    if (left) {
      const bool rest = left >> lane & 1;
      for (int b = 0; (kRows >> b) > 1; ++b) {
        const bool one = (d >> b) & 1;
        const uint64_t v = __builtin_amdgcn_ballot_w64(one);
        left &= one ? v : ~v;
      }
      if (rest) same = left;
    }
    return same;
  };
  // steps of 64 ids for a wave, a multiple of the unrolled loops' (what is past n counts nowhere)
  const int64_t steps = (n + kThreads * kPlaceUnroll - 1) / (kThreads * kPlaceUnroll) * kPlaceUnroll;
  const int64_t lo = w * steps * 64;
#pragma unroll
  for (int i = 0; i < kRows / 64; ++i) count[w * kRows + i * 64 + lane] = 0;
  const uint64_t lower = (1ull << lane) - 1;
  uint32_t below = 0;
  int64_t listed = 0;
  for (int64_t j = 0; j < steps; j += kPlaceUnroll) {
    const int64_t first = lo + j * 64;
    if (first >= n) break;
    I id[kPlaceUnroll];
    const bool full = first + 64 * kPlaceUnroll <= n;
    if (full) {
#pragma unroll
      for (int u = 0; u < kPlaceUnroll; ++u) id[u] = ids[first + u * 64 + lane];
    } else {
#pragma unroll
      for (int u = 0; u < kPlaceUnroll; ++u) id[u] = first + u * 64 + lane < n ? ids[first + u * 64 + lane] : 0;
    }
#pragma unroll
    for (int u = 0; u < kPlaceUnroll; ++u) {
      uint32_t owner = (static_cast<uint32_t>(id[u]) - start_lo) & mask;
      if (!full && first + u * 64 + lane >= n) owner = ~0u;  // nobody's
      below += owner < me;
      const bool own = owner == me;
      const uint64_t all = __builtin_amdgcn_ballot_w64(own);
      if (!all) continue;
      const uint32_t d = counter_of(id[u]);
      // many at once are mostly of one counter, where their additions would wait for each other
      const uint64_t same = __popcll(all) > kCrowd ? peers(all, d) : 0;
      if (own) {
        if (!same) atomicAdd(&count[w * kRows + d], 1u);
        else if (!(same & lower)) atomicAdd(&count[w * kRows + d], static_cast<uint32_t>(__popcll(same)));
        const int64_t at = listed + __popcll(all & lower);
        if (at < kList) list[w][at] = d << 22 | static_cast<uint32_t>((j + u) * 64 + lane);
      }
      listed += __popcll(all);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) below += __shfl_xor(below, off, 64);
  if (lane == 0) wave_sum[0][w] = below;
  __syncthreads();
  // exclusive scan over (row, wave), from the number of lower workgroups' ids on
  uint32_t c[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = tid * kEach + i;
    c[i] = count[e % kWaves * kRows + e / kWaves];
    sum += c[i];
  }
  uint32_t incl = sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t v = __shfl_up(incl, off, 64);
    if (lane >= off) incl += v;
  }
  if (lane == 63) wave_sum[1][w] = incl;
  __syncthreads();
  uint32_t place = incl - sum;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) place += wave_sum[0][i] + (i < w ? wave_sum[1][i] : 0);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int e = tid * kEach + i;
    count[e % kWaves * kRows + e / kWaves] = place;
    place += c[i];
  }
  __syncthreads();
  // places the lanes' own ids, `d` their counters, `at` their indexes
  auto put = [&](bool own, uint32_t d, int64_t at) {
    const uint64_t same = peers(__builtin_amdgcn_ballot_w64(own), d);
    if (own) {
      const uint32_t before = static_cast<uint32_t>(__popcll(same & lower)), to = count[w * kRows + d];
      keep_order();
      if (before == 0) count[w * kRows + d] = to + static_cast<uint32_t>(__popcll(same));
      keep_order();
      const uint32_t row = d == kRows - 1u ? ~0u : d << shift | me;
      sorted[to + before] = static_cast<uint64_t>(row) << 32 | static_cast<uint32_t>(at);
    }
  };
  if (listed <= kList && steps * 64 <= 1 << 22) {
    for (int64_t i = 0; i < listed; i += 64) {
      const bool own = i + lane < listed;
      const uint32_t e = own ? list[w][i + lane] : 0;
      put(own, e >> 22, lo + (e & ((1u << 22) - 1)));
    }
    return;
  }
  for (int64_t j = 0; j < steps; j += kPlaceUnroll) {
    if (lo + j * 64 >= n) break;
    I id[kPlaceUnroll];
#pragma unroll
    for (int u = 0; u < kPlaceUnroll; ++u) {
      const int64_t i = lo + (j + u) * 64 + lane;
      id[u] = ids[i < n ? i : n - 1];
    }
#pragma unroll
    for (int u = 0; u < kPlaceUnroll; ++u) {
      const int64_t i = lo + (j + u) * 64 + lane;
      put(i < n && ((static_cast<uint32_t>(id[u]) - start_lo) & mask) == me, counter_of(id[u]), i);
    }
  }
}

// ------------------------------------------------------------------ gradient
__device__ __forceinline__ int64_t partial_stride(int E) { return (E + 3) & ~3; }

// out = scale a, or scale a + old
template <typename T, bool kAligned>
__device__ __forceinline__ void grad_store(void* out, int64_t at, int64_t left, float (&a)[kFull<T>], float scale,
                                           bool accumulate, const uint4& old) {
  float o[kFull<T>];
  unpackv<T, kFull<T>>(old, o);
#pragma unroll
  for (int k = 0; k < kFull<T>; ++k) {
    a[k] *= scale;
    if (accumulate) a[k] += o[k];
  }
  store_row<T, kAligned, false>(out, at, left, packv<T, kFull<T>>(a));
}
template <typename T, bool kAligned>
__device__ __forceinline__ void grad_store(void* out, int64_t at, int64_t left, float (&a)[kFull<T>], float scale,
                                           bool accumulate) {
  uint4 old = make_uint4(0, 0, 0, 0);
  if (accumulate) old = load_row<T, kAligned, false>(out, at, left);
  grad_store<T, kAligned>(out, at, left, a, scale, accumulate, old);
}

// Few ids: a wave per table row and stretch of 64 V columns. Rows without an id are cleared (or left
// alone when adding), so that this is the gradient's only launch.
constexpr int kDirectWaves = 4;
constexpr int kDirectUnroll = 8;
template <typename T, bool kAligned>
__global__ __launch_bounds__(kDirectWaves * 64) void embed_grad_direct_kernel(
    int64_t block0, EmbedIds ids, const void* __restrict__ dy, void* __restrict__ out, int E, float scale,
    bool accumulate) {
  constexpr int V = kFull<T>;
  const int lane = threadIdx.x & 63;
  const int64_t row = (block0 + blockIdx.x) * kDirectWaves + (threadIdx.x >> 6);
  if (row >= ids.rows) return;
  const int c = (blockIdx.y * 64 + lane) * V;
  const bool ok = c < E;
  const int n = static_cast<int>(ids.n);
  float a[V];
#pragma unroll
  for (int k = 0; k < V; ++k) a[k] = 0.f;
  bool any = false;
#pragma unroll 2
  for (int i0 = 0; i0 < n; i0 += 64) {
    uint64_t own = __ballot(i0 + lane < n && ids.ids.at(i0 + lane) - ids.start == row);
    any |= own != 0;
    while (own) {
      uint4 r[kDirectUnroll];
      int got = 0;
#pragma unroll
      for (int u = 0; u < kDirectUnroll; ++u) {
        if (!own) break;
        const int t = i0 + __builtin_ctzll(own);
        own &= own - 1;
        if (ok) r[u] = load_row<T, kAligned, false>(dy, static_cast<int64_t>(t) * E + c, E - c);
        ++got;
      }
#pragma unroll
      for (int u = 0; u < kDirectUnroll; ++u) {
        if (u >= got || !ok) break;
        float x[V];
        unpackv<T, V>(r[u], x);
#pragma unroll
        for (int k = 0; k < V; ++k) a[k] += x[k];
      }
    }
  }
  if (ok && (any || !accumulate)) grad_store<T, kAligned>(out, row * E + c, E - c, a, scale, accumulate);
}

// Workgroup x takes sorted entries [x K, (x + 1) K), K <= 64, workgroup y a stretch of columns. Every
// wave holds the range's entries in its lanes, so all row addresses are known from the start; the
// next rows' loads (and, when adding, of the table rows that end among them) leave before the present
// ones are added. partial holds two rows a workgroup: 0 the sum of a token that began in an earlier
// range (its "head"), 1 of one that began here and goes on (its "tail").
constexpr int kGradUnroll = 8;
template <typename T, bool kAligned, bool kAdd>
__global__ __launch_bounds__(256) void embed_grad_kernel(int64_t block0, const uint64_t* __restrict__ sorted,
                                                         const void* __restrict__ dy, void* out,
                                                         float* __restrict__ partial, int64_t n, int E, int K,
                                                         float scale) {
  constexpr int V = kFull<T>;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  const bool ok = c < E;
  const int64_t x = block0 + blockIdx.x, lo = x * K;
  const int cnt = static_cast<int>(n - lo < K ? n - lo : K);
  const int64_t ps = partial_stride(E);
  float* head = partial + x * 2 * ps;
  const int lane = threadIdx.x & 63;
  const uint64_t entry = sorted[lo + (lane < cnt ? lane : cnt - 1)];
  const int before = lo > 0 ? row_of(sorted[lo - 1]) : -1;
  const int after = lo + cnt < n ? row_of(sorted[lo + cnt]) : -1;
  const int row_l = row_of(entry);
  const uint32_t tok_l = static_cast<uint32_t>(entry);
  auto row_at = [&](int e) { return e < cnt ? __builtin_amdgcn_readlane(row_l, e) : after; };
  bool open = before == row_at(0);
  float a[V];
#pragma unroll
  for (int k = 0; k < V; ++k) a[k] = 0.f;
  struct Batch {
    uint4 dy[kGradUnroll], old[kAdd ? kGradUnroll : 1];
  };
  // no branches around the rows' loads, so that a wait for one batch leaves the next one in flight:
  // past the end the last entry's row again, lanes past E (their vectors' values are not used) column 0
  const int col = ok ? c : 0;
  auto load = [&](Batch& r, int e) {
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u) {
      const uint32_t tok = __builtin_amdgcn_readlane(tok_l, e + u);
      r.dy[u] = load_row<T, kAligned, true>(dy, static_cast<int64_t>(tok) * E + col, E - col);
    }
    if constexpr (kAdd) {
#pragma unroll
      for (int u = 0; u < kGradUnroll; ++u) {
        if (e + u >= cnt) break;
        const int row = row_at(e + u);
        if (ok && row >= 0 && row != row_at(e + u + 1))
          r.old[u] = load_row<T, kAligned, false>(out, static_cast<int64_t>(row) * E + c, E - c);
      }
    }
  };
  auto add = [&](const Batch& now, int e) {
#pragma unroll
    for (int u = 0; u < kGradUnroll; ++u) {
      if (e + u >= cnt) break;
      const int row = row_at(e + u);
      if (row < 0) {  // ids without a row
        open = false;
        continue;
      }
      if (ok) {
        float x[V];
        unpackv<T, V>(now.dy[u], x);
#pragma unroll
        for (int k = 0; k < V; ++k) a[k] += x[k];
      }
      const bool last = e + u + 1 == cnt, ends = row != row_at(e + u + 1);
      if (!ends && !last) continue;
      // the token ends here, or goes on in the next range
      if (ok) {
        if (open || !ends) {
          float* to = open ? head : head + ps;
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (kAligned || c + k < E) to[c + k] = a[k];
        } else {
          grad_store<T, kAligned>(out, static_cast<int64_t>(row) * E + c, E - c, a, scale, kAdd,
                                  now.old[kAdd ? u : 0]);
        }
      }
#pragma unroll
      for (int k = 0; k < V; ++k) a[k] = 0.f;
      open = false;
    }
  };
  Batch now, then;
  load(now, 0);
  int e = 0;
  for (; e + kGradUnroll < cnt; e += kGradUnroll) {
    load(then, e + kGradUnroll);
    add(now, e);
    now = then;
  }
  add(now, e);
}

// Joins the tokens that cross ranges: the workgroup in whose range a token begins adds the heads of
// the following ranges to its tail. 4 waves take every fourth range, 256 columns a workgroup.
constexpr int kJoinWaves = 4;
template <typename T>
__global__ __launch_bounds__(kJoinWaves * 64) void embed_join_kernel(int64_t block0,
                                                                     const uint64_t* __restrict__ sorted,
                                                                     const float* __restrict__ partial,
                                                                     void* __restrict__ out, int64_t n, int E,
                                                                     int K, float scale, bool accumulate) {
  __shared__ float4 red[kJoinWaves][64];
  const int64_t x = block0 + blockIdx.x, lo = x * K, hi = lo + K;
  if (hi >= n) return;
  const int row = row_of(sorted[hi - 1]), next = row_of(sorted[hi]), first = row_of(sorted[lo]);
  const int before = row_of(sorted[lo > 0 ? lo - 1 : 0]);
  if (row < 0 || next != row) return;                   // ends here
  if (lo > 0 && first == row && before == row) return;  // began earlier
  // the last range that begins with the token (they follow each other): 64 ranges a step, since a step
  // costs a trip to memory, 64 times as far apart while all have it, and back
  const int64_t nb = (n + K - 1) / K;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int64_t last = x;
  for (int64_t apart = 1; apart;) {
    const int64_t at = last + (lane + 1) * apart;
    const int with = __popcll(__builtin_amdgcn_ballot_w64(at < nb && row_of(sorted[at < nb ? at * K : 0]) == row));
    last += with * apart;
    apart = with == 64 ? apart * 64 : apart / 64;
  }
  const int c = (blockIdx.y * 64 + lane) * 4;
  const int64_t ps = partial_stride(E);
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < E) {
#pragma unroll 8
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
    const int64_t at = static_cast<int64_t>(row) * E + c + k;
    Elem<T>::put(out, at, accumulate ? v[k] * scale + Elem<T>::get(out, at) : v[k] * scale);
  }
}

// ------------------------------------------------------------------ position gradient
// Column sums of dy [B][N]: a lane takes V columns, the workgroup's waves split the batch and join
// in a fixed order.
constexpr int kSumUnroll = 8;
template <typename T, bool kAligned>
__global__ __launch_bounds__(1024) void batch_sum_kernel(int64_t block0, const void* __restrict__ dy,
                                                         void* __restrict__ out,
                                                         int64_t B, int64_t N, bool accumulate) {
  constexpr int V = kFull<T>;
  extern __shared__ float red[];  // [waves][64][V]
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int64_t c = ((block0 + blockIdx.x) * 64 + lane) * V;
  float a[V];
#pragma unroll
  for (int k = 0; k < V; ++k) a[k] = 0.f;
  if (c < N) {
    int64_t b = w;
    for (; b + (kSumUnroll - 1) * waves < B; b += static_cast<int64_t>(waves) * kSumUnroll) {
      uint4 r[kSumUnroll];
#pragma unroll
      for (int u = 0; u < kSumUnroll; ++u) r[u] = load_row<T, kAligned, false>(dy, (b + u * waves) * N + c, N - c);
#pragma unroll
      for (int u = 0; u < kSumUnroll; ++u) {
        float x[V];
        unpackv<T, V>(r[u], x);
#pragma unroll
        for (int k = 0; k < V; ++k) a[k] += x[k];
      }
    }
    for (; b < B; b += waves) {
      float x[V];
      unpackv<T, V>(load_row<T, kAligned, false>(dy, b * N + c, N - c), x);
#pragma unroll
      for (int k = 0; k < V; ++k) a[k] += x[k];
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
  if (c < N) grad_store<T, kAligned>(out, c, N - c, a, 1.f, accumulate);
}

template <typename T, typename F>
void dispatch_a(bool aligned, F&& f) {
  if (aligned) f(T{}, BTag<true>{});
  else f(T{}, BTag<false>{});
}
template <typename F>
void dispatch_ta(TDtype dt, bool aligned, F&& f) {
  switch (dt) {
    case TDtype::kBF16: dispatch_a<BF16>(aligned, f); break;
    case TDtype::kF16: dispatch_a<F16>(aligned, f); break;
    default: dispatch_a<F32>(aligned, f); break;
  }
}

// Sorted entries a workgroup takes: enough workgroups to fill the chip, few partial rows (32k ids,
// E = 1024, bf16, both kernels: 8 entries 42 us, 16 38 us, 32 33 us, 64 36 us).
int grad_range(int64_t n) { return n >= 16384 ? 32 : (n >= 4096 ? 16 : 8); }

// Whether a wave per table row is quicker than the sort and its two further launches. It looks through
// n ids for every row, so the answer depends on both (kernels alone, ids spread out: 256 ids for 512 rows
// of 128 fp32 9 against 12 us, 512 ids 14 against 13; 50304 rows of 1024 bf16, 128 ids 21 against 24,
// 256 ids 28 against 23). All ids the same is the sort's better case: 256 of them 31 against 13 us.
bool direct(int64_t n, int64_t rows) { return n <= 128 || (n <= 256 && rows <= 4096); }

// f(first workgroup, workgroups) for the launches that `blocks` workgroups take: HIP refuses 2^32
// threads and more in one.
constexpr int64_t kMaxBlocks = 1 << 21;
template <typename F>
void for_blocks(int64_t blocks, F&& f) {
  for (int64_t b = 0; b < blocks; b += kMaxBlocks)
    f(b, static_cast<unsigned>(blocks - b < kMaxBlocks ? blocks - b : kMaxBlocks));
}

int64_t partial_floats(int64_t n, int E) {
  const int64_t K = grad_range(n);
  return (n + K - 1) / K * 2 * ((E + 3) & ~3);
}
}  // namespace

void embed_fwd(TDtype dt, bool aligned, const EmbedIds& ids, const void* table, int64_t stride,
               const EmbedPos& pos, float scale, void* out, int E, hipStream_t st) {
  if (ids.n == 0 || E == 0) return;
  dispatch_ta(dt, aligned, [&](auto t, auto a) {
    using T = decltype(t);
    constexpr int V = kFull<T>;
    constexpr bool A = decltype(a)::value;
    const int64_t nv = (E + V - 1) / V;
    // one pass of the workgroup's unrolled loop, as long as that leaves 1024 workgroups, and rows enough
    // for one launch
    int64_t r = kFwdBlock * kFwdUnroll / nv;
    if (r > ids.n / 1024) r = ids.n / 1024;
    if (r <= ids.n / kMaxBlocks) r = ids.n / kMaxBlocks + 1;
    auto* kernel = ids.n * E * kElem<T> >= kStreamBytes ? embed_fwd_kernel<T, A, true> : embed_fwd_kernel<T, A, false>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((ids.n + r - 1) / r)), dim3(kFwdBlock), 0, st, ids, table,
                       stride, pos, scale, out, E, static_cast<int>(r));
  });
}

// The workspace: the sorted entries, the partial rows.
int64_t embed_grad_workspace(int64_t n, int64_t rows, int E) {
  return direct(n, rows) ? 0 : (n + 1) / 2 * 16 + partial_floats(n, E) * 4;
}

template <typename I, int kRows, int kWaves>
static void place(const EmbedIds& ids, int shift, uint64_t* sorted, void* clear, int64_t clear_bytes,
                  hipStream_t st) {
  int64_t clearing = (clear_bytes / 16 + kWaves * 64 - 1) / (kWaves * 64);
  if (clearing > 2048) clearing = 2048;
  if (clear_bytes && clearing < 1) clearing = 1;
  hipLaunchKernelGGL((embed_place_kernel<I, kRows, kWaves>), dim3(static_cast<unsigned>((1 << shift) + clearing)),
                     dim3(kWaves * 64), 0, st, static_cast<const I*>(ids.ids.p), ids.n, ids.start, ids.rows, shift,
                     sorted, clear, clear_bytes);
}
template <typename I>
static void place(const EmbedIds& ids, uint64_t* sorted, void* clear, int64_t clear_bytes, hipStream_t st) {
  // a workgroup per CU, with counters for 255 or 1023 rows; more workgroups past 256k rows
  int shift = 8;
  while ((ids.rows - 1) >> shift >= 1023) ++shift;
  if ((ids.rows - 1) >> shift < 255) place<I, 256, 16>(ids, shift, sorted, clear, clear_bytes, st);
  else place<I, 1024, 8>(ids, shift, sorted, clear, clear_bytes, st);
}

void embed_grad(TDtype dt, bool aligned, const EmbedIds& ids, const void* dy, void* out, int E,
                float scale, bool accumulate, void* workspace, hipStream_t st) {
  const int64_t n = ids.n;
  if (E == 0 || ids.rows == 0) return;
  if (direct(n, ids.rows)) {
    dispatch_ta(dt, aligned, [&](auto t, auto a) {
      using T = decltype(t);
      constexpr int V = kFull<T>;
      constexpr bool A = decltype(a)::value;
      for_blocks((ids.rows + kDirectWaves - 1) / kDirectWaves, [&](int64_t first, unsigned blocks) {
        hipLaunchKernelGGL((embed_grad_direct_kernel<T, A>),
                           dim3(blocks, static_cast<unsigned>((E + 64 * V - 1) / (64 * V))), dim3(kDirectWaves * 64),
                           0, st, first, ids, dy, out, E, scale, accumulate);
      });
    });
    return;
  }
  uint64_t* sorted = static_cast<uint64_t*>(workspace);
  float* partial = reinterpret_cast<float*>(sorted + (n + 1) / 2 * 2);
  const int64_t clear = accumulate ? 0 : ids.rows * E * (dt == TDtype::kF32 ? 4 : 2);
  if (ids.ids.is32) place<int32_t>(ids, sorted, out, clear, st);
  else place<int64_t>(ids, sorted, out, clear, st);
  const int K = grad_range(n);
  const int64_t nb = (n + K - 1) / K;
  dispatch_ta(dt, aligned, [&](auto t, auto a) {
    using T = decltype(t);
    constexpr int V = kFull<T>;
    constexpr bool A = decltype(a)::value;
    const int nv = (E + V - 1) / V;
    const int threads = nv >= 256 ? 256 : (nv + 63) / 64 * 64;
    auto* kernel = accumulate ? embed_grad_kernel<T, A, true> : embed_grad_kernel<T, A, false>;
    for_blocks(nb, [&](int64_t first, unsigned blocks) {
      hipLaunchKernelGGL(kernel, dim3(blocks, static_cast<unsigned>((nv + threads - 1) / threads)), dim3(threads), 0,
                         st, first, sorted, dy, out, partial, n, E, K, scale);
    });
    if (nb == 1) return;
    for_blocks(nb, [&](int64_t first, unsigned blocks) {
      hipLaunchKernelGGL(embed_join_kernel<T>, dim3(blocks, static_cast<unsigned>((E + 255) / 256)),
                         dim3(kJoinWaves * 64), 0, st, first, sorted, partial, out, n, E, K, scale, accumulate);
    });
  });
}

void batch_sum(TDtype dt, bool aligned, const void* dy, void* out, int64_t B, int64_t N,
               bool accumulate, hipStream_t st) {
  if (N == 0) return;
  dispatch_ta(dt, aligned, [&](auto t, auto a) {
    using T = decltype(t);
    constexpr int V = kFull<T>;
    constexpr bool A = decltype(a)::value;
    const int64_t tiles = (N + 64 * V - 1) / (64 * V);
    int waves = 1;  // split the batch where the columns alone do not fill the chip
    while (waves < 16 && waves * 2 <= B && tiles * waves < 4096) waves *= 2;
    for_blocks(tiles, [&](int64_t first, unsigned blocks) {
      hipLaunchKernelGGL((batch_sum_kernel<T, A>), dim3(blocks), dim3(waves * 64),
                         waves > 1 ? static_cast<size_t>(waves) * 64 * V * sizeof(float) : 0, st, first, dy, out, B, N,
                         accumulate);
    });
  });
}
}  // namespace dca
