// What the kernels of the paged cache share: element types, where a token's row lies, argument checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "asg_common.cuh"

namespace asg {
namespace paged {

constexpr int kMaxDim = 256;

inline bool is_wide(int64_t type) { return type == ASG_TYPE_F32 || type == ASG_TYPE_BF16 || type == ASG_TYPE_F16; }
inline bool is_coded(int64_t type) { return type == ASG_TYPE_E4M3 || type == ASG_TYPE_INT8; }
inline int type_bytes(int64_t type) { return type == ASG_TYPE_F32 ? 4 : is_coded(type) ? 1 : 2; }

// Whether every row of a pool, or of token rows, starts on a multiple of `bytes`.
inline bool rows_aligned(const asg_page_pool& p, int item, int bytes) {
  return ((reinterpret_cast<uintptr_t>(p.data) | static_cast<uintptr_t>(p.page_stride * item) |
           static_cast<uintptr_t>(p.token_stride * item) | static_cast<uintptr_t>(p.head_stride * item)) &
          (bytes - 1)) == 0;
}
inline bool rows_aligned(const asg_token_rows& r, int item, int bytes) {
  return ((reinterpret_cast<uintptr_t>(r.data) | static_cast<uintptr_t>(r.token_stride * item) |
           static_cast<uintptr_t>(r.head_stride * item)) & (bytes - 1)) == 0;
}

// Quotients by a number known on the host: n / d for n < 2^31 is the high word of n * multiplier, shifted, with
// multiplier = ceil(2^(31 + l) / d), 2^l >= d: it exceeds 2^(31 + l) / d by less than 1, so n times it is off by less
// than 2^31 / 2^(31 + l) <= 1 / d of a unit, too little to reach the next multiple.
struct Divisor {
  unsigned d, multiplier, shift;
};
inline Divisor divisor_of(unsigned d) {
  Divisor r = {d, 0u, 0u};
  unsigned l = 0;
  while ((1ull << l) < d) ++l;
  if (l > 0) {  // (d = 1 needs none)
    r.multiplier = static_cast<unsigned>(((1ull << (31 + l)) + d - 1) / d);
    r.shift = l - 1;
  }
  return r;
}

// The checks that the three entry points share (host).
inline int check_pools(const asg_page_pool& key_pool, const asg_page_pool& value_pool, int64_t n_pages,
                       int64_t page_size, int64_t n_heads, int64_t head_dim, int64_t wide_type, int64_t cache_type) {
  ASG_REQUIRE(is_wide(wide_type), ASG_EINVAL, "the type of the tokens must be float32, bfloat16 or float16");
  ASG_REQUIRE(is_wide(cache_type) || is_coded(cache_type), ASG_EINVAL, "unknown type of the pages");
  ASG_REQUIRE(n_pages >= 0 && page_size >= 1 && n_heads >= 1 && head_dim >= 1, ASG_EINVAL,
              "n_pages must be non-negative, page_size, heads and head_dim positive");
  ASG_REQUIRE(head_dim <= kMaxDim, ASG_ERANGE, "the paged kernels hold at most 256 features per head");
  ASG_REQUIRE(n_pages <= 2147483647ll && page_size < (1ll << 30) && n_heads <= 65535, ASG_ERANGE,
              "n_pages, page_size or n_heads exceeds the kernel index range");
  ASG_REQUIRE(n_pages == 0 || (key_pool.data != nullptr && value_pool.data != nullptr), ASG_EINVAL,
              "the pages must not be null");
  if (is_coded(cache_type))
    ASG_REQUIRE(n_pages == 0 || (key_pool.scales != nullptr && value_pool.scales != nullptr), ASG_EINVAL,
                "8-bit pages need scales");
  return ASG_OK;
}

#ifdef __CUDACC__

__device__ __forceinline__ unsigned divide(unsigned n, const Divisor& by) {
  return by.d == 1 ? n : __umulhi(n, by.multiplier) >> by.shift;
}

// Storage types and their float32 values.
using F32 = float;
using BF16 = __nv_bfloat16;
using F16 = __half;
struct E4M3 { uint8_t code; };
struct INT8 { int8_t code; };

template <typename T> struct TypeOf;
template <> struct TypeOf<F32> { static constexpr int id = ASG_TYPE_F32; static constexpr bool coded = false; };
template <> struct TypeOf<BF16> { static constexpr int id = ASG_TYPE_BF16; static constexpr bool coded = false; };
template <> struct TypeOf<F16> { static constexpr int id = ASG_TYPE_F16; static constexpr bool coded = false; };
template <> struct TypeOf<E4M3> { static constexpr int id = ASG_TYPE_E4M3; static constexpr bool coded = true; };
template <> struct TypeOf<INT8> { static constexpr int id = ASG_TYPE_INT8; static constexpr bool coded = true; };

__device__ __forceinline__ float to_float(F32 v) { return v; }
__device__ __forceinline__ float to_float(BF16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(F16 v) { return __half2float(v); }
__device__ __forceinline__ float to_float(E4M3 v) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(v.code, __NV_E4M3)));
}
__device__ __forceinline__ float to_float(INT8 v) { return static_cast<float>(v.code); }

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ F32 from_float<F32>(float v) { return v; }
template <> __device__ __forceinline__ BF16 from_float<BF16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ F16 from_float<F16>(float v) { return __float2half_rn(v); }

// N consecutive elements, moved in vectors of up to 32 bytes (the address is a multiple of their size).
template <typename T, int N>
struct Pack {
  static constexpr int kBytes = N * static_cast<int>(sizeof(T));
  static constexpr int kVec = kBytes < 32 ? kBytes : 32;
  alignas(kVec) T v[N];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kVec == 32) {
      uint32_t* r = reinterpret_cast<uint32_t*>(v);
#pragma unroll
      for (int i = 0; i < kBytes / 32; ++i)
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r[8 * i]), "=r"(r[8 * i + 1]), "=r"(r[8 * i + 2]), "=r"(r[8 * i + 3]), "=r"(r[8 * i + 4]),
                       "=r"(r[8 * i + 5]), "=r"(r[8 * i + 6]), "=r"(r[8 * i + 7])
                     : "l"(reinterpret_cast<const uint32_t*>(p) + 8 * i)
                     : "memory");
    } else {
      move(v, p);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kVec == 32) {
      const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
#pragma unroll
      for (int i = 0; i < kBytes / 32; ++i)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<uint32_t*>(p) + 8 * i),
                     "r"(r[8 * i]), "r"(r[8 * i + 1]), "r"(r[8 * i + 2]), "r"(r[8 * i + 3]), "r"(r[8 * i + 4]),
                     "r"(r[8 * i + 5]), "r"(r[8 * i + 6]), "r"(r[8 * i + 7])
                     : "memory");
    } else {
      move(p, v);
    }
  }
  static __device__ __forceinline__ void move(T* to, const T* from) {
    if constexpr (kVec == 16) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
    else if constexpr (kVec == 8) *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(from);
    else if constexpr (kVec == 4) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
    else if constexpr (kVec == 2) *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
    else {
#pragma unroll
      for (int i = 0; i < N; ++i) to[i] = from[i];
    }
  }
};

// The values of a pack; e4m3 is converted two at a time.  (int8 by the conversion instruction, although it runs at an
// eighth of the FMA rate: 65536 tokens of 8 x 128 read as bfloat16 take 71 us, with byte permutes and subtractions 78.)
template <typename T, int N>
__device__ __forceinline__ void to_floats(const Pack<T, N>& p, float (&x)[N]) {
  if constexpr (std::is_same<T, E4M3>::value && N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 v = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(reinterpret_cast<const uint16_t*>(p.v)[i], __NV_E4M3)));
      x[2 * i] = v.x;
      x[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_float(p.v[i]);
  }
}

#endif  // __CUDACC__

}  // namespace paged
}  // namespace asg
