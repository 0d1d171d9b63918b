// Norm of a list of gradients and their clipping, for any number of separate tensors.
//
//   N = sqrt(sum g^2) | sum |g| | max |g|  over all tensors,   g *= min(1, max_norm / (N + 1e-6))
//
// Bound by HBM: the norm reads every gradient once, clipping reads and writes them once more. At 774M
// elements in 436 tensors (GPT-2-large, bf16 and fp32, 1.55 GB) the norm takes 242 us and its joining
// 9 us (6.2 TB/s of reads), the scaling 491 us (6.3 TB/s). Tensors are cut into
// chunks of one size, a workgroup a chunk, and up to kMaxTensors tensors go by value in the arguments of
// one launch: no table to copy to the device, nothing to keep alive, graph-capturable.
// Sums are held in 64 bits (gradients of 1e-25 or 1e+25 neither vanish nor overflow when squared, and
// the fp64 rate is far above what the loads need) and joined in a fixed order, without atomics.
#include "grad_norm_api.h"

#include "rowvec.h"

namespace dca {
namespace {

constexpr int kNormBlock = 256;
constexpr int kMaxTensors = 192;  // 192 x 20 bytes of arguments; a launch holds 4 KB of them
constexpr int kUnroll = 4;

struct TensorTable {
  uint64_t p[kMaxTensors];
  int64_t n_dt[kMaxTensors];       // elements * 4 + type
  uint32_t first[kMaxTensors];     // its first workgroup in this launch
  int count;
  int64_t chunk;                   // elements a workgroup takes
  int64_t partial0;                // partial of the launch's first workgroup
};

struct Piece {
  void* p;
  int64_t lo, hi;
  int dt;
};

// The piece of the list that workgroup `x` takes: the last tensor whose first workgroup is <= x.
__device__ __forceinline__ Piece piece_of(const TensorTable& t, uint32_t x) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.first[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  Piece a;
  // through the global address space: from a plain integer the compiler makes flat accesses
  a.p = (void*)reinterpret_cast<__attribute__((address_space(1))) char*>(t.p[lo]);
  a.dt = static_cast<int>(t.n_dt[lo] & 3);
  const int64_t n = t.n_dt[lo] >> 2;
  a.lo = static_cast<int64_t>(x - t.first[lo]) * t.chunk;
  a.hi = a.lo + t.chunk < n ? a.lo + t.chunk : n;
  return a;
}

// f(element index) for the elements of [lo, hi) before the first 16-byte boundary and after the last
// one, g(first element) for the full vectors between them.
template <typename T, typename F, typename G>
__device__ __forceinline__ void walk(const Piece& a, F&& f, G&& g) {
  const uint64_t at = reinterpret_cast<uint64_t>(a.p) + static_cast<uint64_t>(a.lo) * kElem<T>;
  int64_t body = a.lo + static_cast<int64_t>((16 - at % 16) % 16 / kElem<T>);
  if (body > a.hi) body = a.hi;
  const int64_t vecs = (a.hi - body) / kFull<T>, tail = body + vecs * kFull<T>;
  if (a.lo + threadIdx.x < body) f(a.lo + threadIdx.x);
  for (int64_t i = threadIdx.x; i < vecs; i += kNormBlock * kUnroll) g(body, i, vecs);
  if (tail + threadIdx.x < a.hi) f(tail + threadIdx.x);
}

static_assert(sizeof(TensorTable) + 64 <= 4096, "the arguments of one launch");

template <NormKind kKind>
__device__ __forceinline__ double join(double a, double b) {
  if constexpr (kKind == NormKind::kMax) return (a > b || a != a) ? a : b;  // NaN wins
  else return a + b;
}
template <NormKind kKind>
__device__ __forceinline__ void take(double& s, float v) {
  if constexpr (kKind == NormKind::kL2) s = fma(static_cast<double>(v), static_cast<double>(v), s);
  else if constexpr (kKind == NormKind::kL1) s += static_cast<double>(fabsf(v));
  else s = join<kKind>(s, static_cast<double>(fabsf(v)));
}

// Joins the workgroup's values; valid in thread 0.
template <NormKind kKind>
__device__ __forceinline__ double block_join(double v, double* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = join<kKind>(v, __shfl_xor(v, off, 64));
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) red[w] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < static_cast<int>(blockDim.x >> 6); ++i) v = join<kKind>(v, red[i]);
  return v;
}

template <NormKind kKind, typename T, bool kStream>
__device__ __forceinline__ double piece_norm(const Piece& a) {
  double s[kUnroll] = {};
  walk<T>(
      a, [&](int64_t i) { float v[1]; unpackv<T, 1>(ldv<T, 1>(a.p, i), v); take<kKind>(s[0], v[0]); },
      [&](int64_t body, int64_t i, int64_t vecs) {
        uint4 r[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (i + u * kNormBlock < vecs)
            r[u] = load_row<T, true, kStream>(a.p, body + (i + u * kNormBlock) * kFull<T>, kFull<T>);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          if (i + u * kNormBlock >= vecs) continue;
          float v[kFull<T>];
          unpackv<T, kFull<T>>(r[u], v);
#pragma unroll
          for (int k = 0; k < kFull<T>; ++k) take<kKind>(s[u], v[k]);
        }
      });
#pragma unroll
  for (int u = 1; u < kUnroll; ++u) s[0] = join<kKind>(s[0], s[u]);
  return s[0];
}

template <NormKind kKind, bool kStream>
__global__ __launch_bounds__(kNormBlock) void norm_partial_kernel(TensorTable t, double* __restrict__ partial) {
  __shared__ double red[kNormBlock / 64];
  const Piece a = piece_of(t, blockIdx.x);
  double s;
  if (a.dt == static_cast<int>(TDtype::kBF16)) s = piece_norm<kKind, BF16, kStream>(a);
  else if (a.dt == static_cast<int>(TDtype::kF16)) s = piece_norm<kKind, F16, kStream>(a);
  else s = piece_norm<kKind, F32, kStream>(a);
  s = block_join<kKind>(s, red);
  if (threadIdx.x == 0) partial[t.partial0 + blockIdx.x] = s;
}

template <NormKind kKind>
__global__ __launch_bounds__(1024) void norm_join_kernel(const double* __restrict__ partial, int64_t n,
                                                         float* __restrict__ norm) {
  __shared__ double red[16];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s = join<kKind>(s, partial[i]);
  s = block_join<kKind>(s, red);
  if (threadIdx.x == 0) norm[0] = static_cast<float>(kKind == NormKind::kL2 ? sqrt(s) : s);
}

template <typename T, bool kStream>
__device__ __forceinline__ void piece_scale(const Piece& a, float c) {
  walk<T>(
      a,
      [&](int64_t i) {
        float v[1];
        unpackv<T, 1>(ldv<T, 1>(a.p, i), v);
        v[0] *= c;
        stv<T, 1>(a.p, i, packv<T, 1>(v));
      },
      [&](int64_t body, int64_t i, int64_t vecs) {
        uint4 r[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (i + u * kNormBlock < vecs)
            r[u] = load_row<T, true, kStream>(a.p, body + (i + u * kNormBlock) * kFull<T>, kFull<T>);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          if (i + u * kNormBlock >= vecs) continue;
          float v[kFull<T>];
          unpackv<T, kFull<T>>(r[u], v);
#pragma unroll
          for (int k = 0; k < kFull<T>; ++k) v[k] *= c;
          store_row<T, true, kStream>(a.p, body + (i + u * kNormBlock) * kFull<T>, kFull<T>, packv<T, kFull<T>>(v));
        }
      });
}

// The coefficient in the order of the formula, in fp32; a NaN norm makes every gradient NaN. A
// gradient times 1 is itself, so workgroups of a list within the limit leave it alone.
template <bool kStream>
__global__ __launch_bounds__(kNormBlock) void clip_kernel(TensorTable t, const float* __restrict__ norm,
                                                          float max_norm) {
  const float c = max_norm / (norm[0] + 1e-6f);
  if (c >= 1.f) return;
  const Piece a = piece_of(t, blockIdx.x);
  if (a.dt == static_cast<int>(TDtype::kBF16)) piece_scale<BF16, kStream>(a, c);
  else if (a.dt == static_cast<int>(TDtype::kF16)) piece_scale<F16, kStream>(a, c);
  else piece_scale<F32, kStream>(a, c);
}

// How a list is walked. Lists that do not fit the 256 MB of last-level cache are streamed past it (774M
// elements, bf16: norm 242 against 295 us, scaling 491 against 545 us); from smaller ones the scaling
// finds in it what the norm has read.
struct Walk {
  int64_t norm_chunk;  // elements a workgroup takes: up to 32k, which keeps the norm's partials few
  int64_t clip_chunk;  // the scaling has none to keep: 8k (the list above: 16k 520 us, 2k 515 us)
  bool stream;
};
Walk walk_of(const std::vector<GradTensor>& t) {
  int64_t total = 0, bytes = 0;
  for (const auto& x : t) {
    total += x.n;
    bytes += x.n * (x.dt == TDtype::kF32 ? 4 : 2);
  }
  int64_t c = 2048;  // small lists: workgroups for every CU
  while (c < 32768 && total / c > 2048) c *= 2;
  int64_t clip = c < 8192 ? c : 8192;
  while (total / clip > 1 << 22) clip *= 2;  // HIP refuses launches of 2^32 threads
  return {c, clip, bytes > 256 << 20};
}

// f(table, workgroups) for every launch of the list
template <typename F>
void for_launches(const std::vector<GradTensor>& t, int64_t chunk, F&& f) {
  TensorTable a;
  a.chunk = chunk;
  a.partial0 = 0;
  a.count = 0;
  uint32_t blocks = 0;
  auto flush = [&] {
    if (a.count) f(a, blocks);
    a.partial0 += blocks;
    a.count = 0;
    blocks = 0;
  };
  for (const auto& x : t) {
    if (x.n == 0) continue;
    a.p[a.count] = reinterpret_cast<uint64_t>(x.p);
    a.n_dt[a.count] = x.n * 4 + static_cast<int>(x.dt);
    a.first[a.count++] = blocks;
    blocks += static_cast<uint32_t>((x.n + a.chunk - 1) / a.chunk);
    if (a.count == kMaxTensors || blocks > (1u << 30)) flush();
  }
  flush();
}

template <NormKind kKind>
void grad_norm_kind(const std::vector<GradTensor>& t, double* partial, float* norm, hipStream_t st) {
  const Walk walk = walk_of(t);
  int64_t parts = 0;
  for_launches(t, walk.norm_chunk, [&](const TensorTable& a, uint32_t blocks) {
    auto* kernel = walk.stream ? norm_partial_kernel<kKind, true> : norm_partial_kernel<kKind, false>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kNormBlock), 0, st, a, partial);
    parts += blocks;
  });
  hipLaunchKernelGGL(norm_join_kernel<kKind>, dim3(1), dim3(1024), 0, st, partial, parts, norm);
}
}  // namespace

int64_t grad_norm_workspace(const std::vector<GradTensor>& t) {
  const int64_t c = walk_of(t).norm_chunk;
  int64_t n = 1;
  for (const auto& x : t) n += (x.n + c - 1) / c;
  return n;
}

void grad_norm(const std::vector<GradTensor>& t, NormKind kind, double* partial, float* norm, hipStream_t st) {
  if (kind == NormKind::kL2) grad_norm_kind<NormKind::kL2>(t, partial, norm, st);
  else if (kind == NormKind::kL1) grad_norm_kind<NormKind::kL1>(t, partial, norm, st);
  else grad_norm_kind<NormKind::kMax>(t, partial, norm, st);
}

void grad_clip(const std::vector<GradTensor>& t, const float* norm, float max_norm, hipStream_t st) {
  const Walk walk = walk_of(t);
  for_launches(t, walk.clip_chunk, [&](const TensorTable& a, uint32_t blocks) {
    auto* kernel = walk.stream ? clip_kernel<true> : clip_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kNormBlock), 0, st, a, norm, max_norm);
  });
}
}  // namespace dca
