// Row vectors of 16, 4 or 2 bytes for kernels that take any width and alignment: V elements of
// storage type T, loaded raw (so that unrolled loads are all in flight before the first use) and
// unpacked to fp32. The host picks the widest V that divides the row length, the row strides and
// the base addresses (widest_vec).
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

// Streamed forms, for data past the caches that is not read again soon.
template <typename T, int V>
__device__ __forceinline__ RawVec<T, V> ldv_nt(const void* base, int64_t elem) {
  if constexpr (V * kElem<T> == 16)
    return ldnt16(reinterpret_cast<const typename T::raw*>(base) + elem);
  else
    return ldv<T, V>(base, elem);
}
__device__ __forceinline__ void stnt16(void* p, const uint4& v) {
  const dca_u32x4 r = {v.x, v.y, v.z, v.w};
  __builtin_nontemporal_store(r, static_cast<dca_u32x4*>(p));
}
template <typename T, int V>
__device__ __forceinline__ void stv_nt(void* base, int64_t elem, const RawVec<T, V>& r) {
  if constexpr (V * kElem<T> == 16) stnt16(reinterpret_cast<typename T::raw*>(base) + elem, r);
  else stv<T, V>(base, elem, r);
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
