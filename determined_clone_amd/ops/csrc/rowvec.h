// Vectors of a storage type T for kernels that take any width and alignment: loaded raw (so that
// unrolled loads are all in flight before the first use) and unpacked to fp32.
#pragma once
#include "common.h"

namespace dca {

template <int B> struct RawBytes;
template <> struct RawBytes<16> { using type = uint4; };
template <> struct RawBytes<4> { using type = uint32_t; };
template <> struct RawBytes<2> { using type = uint16_t; };

template <typename T> constexpr int kElem = static_cast<int>(sizeof(typename T::raw));
template <typename T> constexpr int kFull = 16 / kElem<T>;  // elements of a 16-byte vector
template <typename T> constexpr int kHalf = 4 / kElem<T>;   // elements of a 4-byte vector
template <typename T, int V> using RawVec = typename RawBytes<V * kElem<T>>::type;

template <typename T, int V>
__device__ __forceinline__ RawVec<T, V> ldv(const void* base, int64_t elem) {
  return *reinterpret_cast<const RawVec<T, V>*>(reinterpret_cast<const typename T::raw*>(base) + elem);
}
template <typename T, int V>
__device__ __forceinline__ void stv(void* base, int64_t elem, const RawVec<T, V>& r) {
  *reinterpret_cast<RawVec<T, V>*>(reinterpret_cast<typename T::raw*>(base) + elem) = r;
}

// 16-byte vectors of rows of any length and alignment. kAligned: all addresses are multiples of 16
// and `left`, the elements from `elem` to the row's end, is a multiple of the vector's; otherwise the
// address is a multiple of the element's (gfx950 takes such loads and stores as they are) and a row's
// last vector goes element by element, zeros behind it. kStream: past the caches, for data that is
// not read again soon.
template <int kBytes> struct LooseVec;
typedef dca_u32x4 dca_u32x4_2 __attribute__((aligned(2)));
typedef dca_u32x4 dca_u32x4_4 __attribute__((aligned(4)));
template <> struct LooseVec<2> { using type = dca_u32x4_2; };
template <> struct LooseVec<4> { using type = dca_u32x4_4; };
template <typename T, bool kAligned>
using RowPtr = std::conditional_t<kAligned, dca_u32x4, typename LooseVec<kElem<T>>::type>;

template <typename T, bool kAligned, bool kStream>
__device__ __forceinline__ uint4 load_row(const void* base, int64_t elem, int64_t left) {
  const auto* p = reinterpret_cast<const typename T::raw*>(base) + elem;
  if (kAligned || left >= kFull<T>) {
    const auto* q = reinterpret_cast<const RowPtr<T, kAligned>*>(p);
    dca_u32x4 v;
    if constexpr (kStream) v = __builtin_nontemporal_load(q);
    else v = *q;
    return make_uint4(v.x, v.y, v.z, v.w);
  }
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < kFull<T>; ++i) {
    if (i >= left) break;
    if constexpr (kElem<T> == 2) w[i / 2] |= static_cast<uint32_t>(p[i]) << (i % 2 * 16);
    else w[i] = __float_as_uint(p[i]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// (kStream is a template argument also because the compiler would join the two kinds of store of a
// branch into one plain store.)
template <typename T, bool kAligned, bool kStream>
__device__ __forceinline__ void store_row(void* base, int64_t elem, int64_t left, const uint4& r) {
  auto* p = reinterpret_cast<typename T::raw*>(base) + elem;
  if (kAligned || left >= kFull<T>) {
    auto* q = reinterpret_cast<RowPtr<T, kAligned>*>(p);
    const dca_u32x4 v = {r.x, r.y, r.z, r.w};
    if constexpr (kStream) __builtin_nontemporal_store(v, q);
    else *q = v;
    return;
  }
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < kFull<T>; ++i) {
    if (i >= left) break;
    if constexpr (kElem<T> == 2) p[i] = static_cast<uint16_t>(w[i / 2] >> (i % 2 * 16));
    else p[i] = __uint_as_float(w[i]);
  }
}

template <typename T, int V>
__device__ __forceinline__ void unpackv(const RawVec<T, V>& r, float (&v)[V]) {
  if constexpr (std::is_same<T, F32>::value) {
    __builtin_memcpy(v, &r, sizeof(r));
  } else if constexpr (V == 1) {
    v[0] = std::is_same<T, BF16>::value ? __uint_as_float(static_cast<uint32_t>(r) << 16) : h2f(r);
  } else {
    uint32_t w[V / 2];
    __builtin_memcpy(w, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      v[2 * i] = std::is_same<T, BF16>::value ? bf16_lo(w[i]) : h2f(w[i] & 0xffffu);
      v[2 * i + 1] = std::is_same<T, BF16>::value ? bf16_hi(w[i]) : h2f(w[i] >> 16);
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ RawVec<T, V> packv(const float (&v)[V]) {
  RawVec<T, V> r;
  if constexpr (std::is_same<T, F32>::value) {
    __builtin_memcpy(&r, v, sizeof(r));
  } else if constexpr (V == 1) {
    r = std::is_same<T, BF16>::value ? static_cast<uint16_t>(f2bf_bits(v[0])) : f2h(v[0]);
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      w[i] = std::is_same<T, BF16>::value
                 ? pack_bf16x2(v[2 * i], v[2 * i + 1])
                 : static_cast<uint32_t>(f2h(v[2 * i])) | (static_cast<uint32_t>(f2h(v[2 * i + 1])) << 16);
    __builtin_memcpy(&r, w, sizeof(r));
  }
  return r;
}

// An int32 or int64 index array.
struct Index {
  const void* p = nullptr;
  bool is32 = false;
  __device__ __forceinline__ int64_t at(int64_t i) const {
    return is32 ? static_cast<int64_t>(static_cast<const int32_t*>(p)[i]) : static_cast<const int64_t*>(p)[i];
  }
};

// Accumulates the OR of row lengths, strides (elements) and addresses (bytes): the widest of 16, 4
// bytes or one element that divides all of them.
struct WidestVec {
  uint64_t bits = 0;
  int elem;
  explicit WidestVec(int elem_bytes) : elem(elem_bytes) {}
  void elems(int64_t n) { bits |= static_cast<uint64_t>(n) * static_cast<uint64_t>(elem); }
  void ptr(const void* p) { bits |= reinterpret_cast<uint64_t>(p); }
  int bytes() const { return bits % 16 == 0 ? 16 : (bits % 4 == 0 ? 4 : elem); }
};

template <bool B>
struct BTag {
  static constexpr bool value = B;
};
template <int V>
struct VTag {
  static constexpr int value = V;
};
// f(T tag, V tag) for a storage type and a vector width in bytes
template <typename T, typename F>
void dispatch_v(int bytes, F&& f) {
  if (bytes == 16) f(T{}, VTag<kFull<T>>{});
  else if (bytes == 4 && kElem<T> < 4) f(T{}, VTag<kHalf<T>>{});
  else f(T{}, VTag<1>{});
}

}  // namespace dca
