// Element types of the language-model operators (fp32, fp16, bf16 storage;
// arithmetic is fp32) and the wave-wide reductions they share.
#pragma once

#include "internal.h"

namespace polar_hip_detail {

// Sixteen bytes of a tensor in one lane's registers.  The pointer type of the
// access says what the address is aligned to -- one element, as rows of an odd
// length begin anywhere -- and the global memory of gfx950 takes 16-byte loads
// and stores there: rows of any length and stride share one code path.
typedef uint32_t Pack __attribute__((ext_vector_type(4)));
typedef uint32_t PackAt2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t PackAt4 __attribute__((ext_vector_type(4), aligned(4)));

typedef float Float2 __attribute__((ext_vector_type(2)));
typedef __bf16 Bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 F16x2 __attribute__((ext_vector_type(2)));

struct TypeF32 {
  using Stored = float;
  static constexpr int kVec = 4; // elements in a Pack
  static constexpr int kOrderBits = 20; // leading bits of an fp32 that tell values apart well enough to bound them
  using At = PackAt4;
  __device__ static float widen(float v) { return v; }
  __device__ static float narrow(float v) { return v; }
  __device__ static void unpack(Pack p, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t word = p[i]; // a bit cast of the element itself would read the vector's first one
      x[i] = __builtin_bit_cast(float, word);
    }
  }
  __device__ static Pack pack(const float* x) {
    Pack p;
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __builtin_bit_cast(uint32_t, x[i]);
    return p;
  }
};

struct TypeF16 {
  using Stored = _Float16;
  static constexpr int kVec = 8;
  static constexpr int kOrderBits = 20; // sign, eight bits of exponent, ten of mantissa: all there is
  using At = PackAt2;
  __device__ static float widen(_Float16 v) { return static_cast<float>(v); }
  __device__ static _Float16 narrow(float v) { return static_cast<_Float16>(v); } // to nearest, ties to even
  __device__ static void unpack(Pack p, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t word = p[i];
      const F16x2 h = __builtin_bit_cast(F16x2, word);
      x[2 * i] = static_cast<float>(h.x);
      x[2 * i + 1] = static_cast<float>(h.y);
    }
  }
  __device__ static Pack pack(const float* x) {
    Pack p;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      p[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((Float2{x[2 * i], x[2 * i + 1]}), F16x2));
    return p;
  }
};

struct TypeBF16 {
  using Stored = __bf16;
  static constexpr int kVec = 8;
  static constexpr int kOrderBits = 16; // all there is
  using At = PackAt2;
  __device__ static float widen(__bf16 v) { return static_cast<float>(v); }
  __device__ static __bf16 narrow(float v) { return static_cast<__bf16>(v); } // to nearest, ties to even
  __device__ static void unpack(Pack p, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __builtin_bit_cast(float, p[i] << 16);
      x[2 * i + 1] = __builtin_bit_cast(float, p[i] & 0xffff0000u);
    }
  }
  __device__ static Pack pack(const float* x) {
    Pack p;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      p[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((Float2{x[2 * i], x[2 * i + 1]}), Bf16x2));
    return p;
  }
};

// A Pack of row `row` from element c on; elements at and behind `cols` read as
// `pad` (given as stored) and are not touched in memory.
template <typename T, bool kStream = true>
__device__ __forceinline__ Pack loadPack(const typename T::Stored* row, uint64_t c, uint64_t cols,
                                         typename T::Stored pad) {
  if (c + T::kVec <= cols) {
    const typename T::At* at = reinterpret_cast<const typename T::At*>(row + c);
    if constexpr (kStream)
      return __builtin_nontemporal_load(at);
    else
      return *at;
  }
  typename T::Stored v[T::kVec];
#pragma unroll
  for (int i = 0; i < T::kVec; ++i) v[i] = c + i < cols ? row[c + i] : pad;
  return __builtin_bit_cast(Pack, v);
}

template <typename T>
__device__ __forceinline__ void storePack(typename T::Stored* row, uint64_t c, uint64_t cols, const float* x) {
  if (c + T::kVec <= cols) {
    __builtin_nontemporal_store(T::pack(x), reinterpret_cast<typename T::At*>(row + c));
  } else {
#pragma unroll
    for (int i = 0; i < T::kVec; ++i)
      if (c + i < cols) row[c + i] = T::narrow(x[i]);
  }
}

// kCount consecutive elements of a parameter vector as fp32; `fill` where the
// vector is absent (null) and behind its end.
template <typename P, int kCount>
__device__ __forceinline__ void loadParams(const typename P::Stored* v, uint64_t c, uint64_t cols, float fill, float* out) {
  static_assert(kCount % P::kVec == 0, "whole packs");
  if (v != nullptr && c + kCount <= cols) {
#pragma unroll
    for (int k = 0; k < kCount / P::kVec; ++k)
      P::unpack(*reinterpret_cast<const typename P::At*>(v + c + k * P::kVec), out + k * P::kVec);
  } else {
#pragma unroll
    for (int i = 0; i < kCount; ++i) out[i] = v != nullptr && c + i < cols ? P::widen(v[c + i]) : fill;
  }
}

// ---- wave-wide reductions -------------------------------------------------------
// Data-parallel-primitive moves: neighbours, halves and rows of sixteen lanes are
// exchanged inside the vector ALU (no LDS round trip); the order of the additions
// is fixed by the lane numbers.  The result is in every lane (it comes back through
// a scalar register).
template <int kControl, int kRowMask = 0xf>
__device__ __forceinline__ float dppMove(float fill, float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, fill), __builtin_bit_cast(int, v),
                                                               kControl, kRowMask, 0xf, false));
}
__device__ __forceinline__ float lane63(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ float waveSum(float v) {
  v += dppMove<0xb1>(0.0f, v);       // lane ^ 1
  v += dppMove<0x4e>(0.0f, v);       // lane ^ 2
  v += dppMove<0x141>(0.0f, v);      // mirrored within 8
  v += dppMove<0x140>(0.0f, v);      // mirrored within 16: each row holds its sum
  v += dppMove<0x142, 0xa>(0.0f, v); // row 0 into 1, row 2 into 3
  v += dppMove<0x143, 0xc>(0.0f, v); // lane 31 into rows 2 and 3
  return lane63(v);
}
__device__ __forceinline__ float waveMax(float v) { // a NaN is passed over unless all are
  v = fmaxf(v, dppMove<0xb1>(v, v));
  v = fmaxf(v, dppMove<0x4e>(v, v));
  v = fmaxf(v, dppMove<0x141>(v, v));
  v = fmaxf(v, dppMove<0x140>(v, v));
  v = fmaxf(v, dppMove<0x142, 0xa>(v, v));
  v = fmaxf(v, dppMove<0x143, 0xc>(v, v));
  return lane63(v);
}

// ---- host-side checks -------------------------------------------------------------
inline bool knownType(int type) {
  return type == POLAR_HIP_F32 || type == POLAR_HIP_F16 || type == POLAR_HIP_BF16;
}
inline uint64_t sizeOf(int type) { return type == POLAR_HIP_F32 ? 4 : 2; }
inline bool alignedTo(const void* p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// rows x stride elements of `size` bytes have addresses that 63 bits hold
inline bool addressable(uint64_t rows, uint64_t stride, uint64_t size) {
  uint64_t n = 0;
  return !__builtin_mul_overflow(rows, stride, &n) && !__builtin_mul_overflow(n, size, &n) && n < (1ull << 63);
}

} // namespace polar_hip_detail
