// Loads, stores and small helpers shared by the operators of nn.h.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.h"
#include "nn.h"

namespace xgbb::nn {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive values moved as one access of up to 16 bytes each. The
// address has to be a multiple of min(32, N * sizeof(T)).
template <class T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack {
  T v[N];
  __device__ __forceinline__ float f(int i) const { return to_f32(v[i]); }
};
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load(const T* p) {
  return *reinterpret_cast<const Pack<T, N>*>(p);
}
template <class T, int N>
__device__ __forceinline__ void store(T* p, const float (&f)[N]) {
  Pack<T, N> o;
#pragma unroll
  for (int i = 0; i < N; ++i) o.v[i] = from_f32<T>(f[i]);
  *reinterpret_cast<Pack<T, N>*>(p) = o;
}

// The same in global memory, where eight floats are one access of 32 bytes.
template <class T, int N>
__device__ __forceinline__ void store_global(T* p, const float (&f)[N]) {
  if constexpr (sizeof(T) * N == 32) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]),
                 "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
                 : "memory");
  } else {
    store<T, N>(p, f);
  }
}

// Shared memory to global memory behind the threads' backs, both and the size
// in multiples of 16 bytes. What the threads wrote to the source has to be
// fenced before, and the issuing thread waits for its copies before it ends.
__device__ __forceinline__ void bulk_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void bulk_store(void* to, const void* from, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to),
               "r"(uint32_t(__cvta_generic_to_shared(from))), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_wait_all() {
  asm volatile("cp.async.bulk.commit_group;\ncp.async.bulk.wait_group 0;" ::: "memory");
}

// Two float32 operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)),
        "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// 16 bytes of T as float pairs and back.
template <class T>
__device__ __forceinline__ void unpack16(const uint4& p, float2 (&f)[8 / sizeof(T)]) {
  const uint32_t w[4] = {p.x, p.y, p.z, p.w};
  if constexpr (sizeof(T) == 4) {
    f[0] = make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
    f[1] = make_float2(__uint_as_float(w[2]), __uint_as_float(w[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, __half>)
        f[i] = __half22float2(reinterpret_cast<const __half2&>(w[i]));
      else
        f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
  }
}
template <class T>
__device__ __forceinline__ uint4 pack16(const float2 (&f)[8 / sizeof(T)]) {
  uint4 p;
  uint32_t w[4];
  if constexpr (sizeof(T) == 4) {
    p = make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x),
                   __float_as_uint(f[1].y));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __float22half2_rn(f[i]);
        w[i] = reinterpret_cast<const uint32_t&>(h);
      } else {
        const __nv_bfloat162 h = __float22bfloat162_rn(f[i]);
        w[i] = reinterpret_cast<const uint32_t&>(h);
      }
    }
    p = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return p;
}

// 2 H values of P as float pairs, from an address that is a multiple of their
// size (32 bytes for eight floats).
template <class P, int H>
__device__ __forceinline__ void load_pairs(const P* p, float2 (&f)[H]) {
  if constexpr (sizeof(P) * H == 16) {
    asm("ld.global.nc.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=f"(f[0].x), "=f"(f[0].y), "=f"(f[1].x), "=f"(f[1].y), "=f"(f[2].x), "=f"(f[2].y), "=f"(f[3].x),
          "=f"(f[3].y)
        : "l"(p));
  } else {
    unpack16<P>(*reinterpret_cast<const uint4*>(p), f);
  }
}

// An even number of values as float pairs.
template <class T, int VE>
__device__ __forceinline__ float2 pair_of(const Pack<T, VE>& p, int i) {
  if constexpr (sizeof(T) == 4) {
    return make_float2(p.f(2 * i), p.f(2 * i + 1));
  } else {
    const uint32_t w = reinterpret_cast<const uint32_t*>(&p)[i];
    if constexpr (std::is_same_v<T, __half>) return __half22float2(reinterpret_cast<const __half2&>(w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
}

// A row's values summed up, in pairs of float32 where they are even in number.
template <class T, int VE>
struct Sum {
  static constexpr bool kPairs = VE % 2 == 0;
  float2 two[kPairs ? VE / 2 : 1];
  float one;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (float2& v : two) v = make_float2(0.0f, 0.0f);
    one = 0.0f;
  }
  template <bool SCALED>
  __device__ __forceinline__ void add(const Pack<T, VE>& p, float f) {
    if constexpr (kPairs) {
#pragma unroll
      for (int e = 0; e < VE / 2; ++e) {
        const float2 v = pair_of<T, VE>(p, e);
        two[e] = SCALED ? fma2(make_float2(f, f), v, two[e]) : add2(two[e], v);
      }
    } else {
      static_assert(kPairs || VE == 1, "one value or pairs");
      one = SCALED ? fmaf(f, p.f(0), one) : one + p.f(0);
    }
  }
  __device__ __forceinline__ void get(float (&f)[VE]) const {
#pragma unroll
    for (int e = 0; e < VE; ++e) f[e] = !kPairs ? one : e % 2 ? two[e / 2].y : two[e / 2].x;
  }
};

// Copies 16 bytes into shared memory behind the thread's back; a thread that
// waits for its own copies needs no barrier to read them.
__device__ __forceinline__ void copy_async16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(uint32_t(__cvta_generic_to_shared(to))), "l"(from)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most N of the thread's last groups are under way.
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Division of 32-bit numbers by an invariant divisor: with s = ceil(log2 d)
// and m = floor(2^32 (2^s - d) / d) + 1, n / d = (mulhi(n, m) + n) >> s, the
// sum in 33 bits (Granlund and Montgomery, "Division by invariant integers
// using multiplication", 1994).
struct FastDiv {
  uint32_t d, m, s;
  FastDiv() : d(1), m(1), s(0) {}
  explicit FastDiv(uint32_t divisor) : d(divisor), s(0) {
    while (s < 32 && (1ull << s) < divisor) ++s;
    m = uint32_t((((1ull << s) - divisor) << 32) / divisor + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return uint32_t((uint64_t(__umulhi(n, m)) + n) >> s);
  }
};

__device__ __forceinline__ int64_t load_token(const void* data, bool wide, int64_t at) {
  return wide ? static_cast<const int64_t*>(data)[at] : int64_t(static_cast<const int32_t*>(data)[at]);
}

// Whether every row starts at a multiple of n values' bytes, or of 32.
inline bool row_aligned(const void* p, int64_t stride, uint64_t rows, size_t size, uint64_t n) {
  const size_t b = n * size < 32 ? n * size : 32;
  return reinterpret_cast<uintptr_t>(p) % b == 0 && (rows <= 1 || (stride * int64_t(size)) % int64_t(b) == 0);
}

// log2 of the lanes that own a row of `pieces` or a tile of it: up to 8 lanes as
// many as it takes, else as many of 8, 16 and 32 as leave no more lanes idle in
// the last tile than 8 would. (33 columns in two tiles of 32 lanes took bags of
// 100 tokens 137 us where five tiles of 8 take 104.) And as many as leave no more
// tiles than a grid has in y, whatever lanes are idle.
inline int lanes_log2(uint64_t pieces) {
  constexpr uint64_t kTiles = 65535;
  int lg = 0;
  while (lg < 3 && (1ull << lg) < pieces) ++lg;
  while (lg >= 3 && lg < 5 && (((pieces + 7) / 8 * 8) % (2ull << lg) == 0 || pieces > kTiles << lg)) ++lg;
  return lg;
}

// Lets a kernel be launched with `shared` bytes of dynamic shared memory. The
// limit belongs to the kernel on its device and not to one launch, so every call
// sets the same one, the `most` that any launch of the kernel asks for: another
// host thread's launch may come between this and the caller's.
template <class... Params>
void allow_shared(void (*kernel)(Params...), size_t shared, size_t most) {
  require(shared <= most, "a launch asks for more shared memory than its kernel allows");
  if (shared > 40 * 1024)
    XGBB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(most)));
}

inline unsigned blocks_for(uint64_t work, uint64_t per_block) {
  return unsigned((work + per_block - 1) / per_block);
}

// Calls f with a null pointer of the type that a dtype code stands for.
template <class F>
void with_type(int type, F&& f) {
  if (type == kF32) f(static_cast<float*>(nullptr));
  else if (type == kF16) f(static_cast<__half*>(nullptr));
  else f(static_cast<__nv_bfloat16*>(nullptr));
}
// The same for a pair (a, b): equal, or one of them float.
template <class F>
void with_types(int a, int b, F&& f) {
  with_type(a, [&](auto* pa) {
    if (a == b) f(pa, pa);
    else if constexpr (std::is_same_v<decltype(pa), float*>) with_type(b, [&](auto* pb) { f(pa, pb); });
    else f(pa, static_cast<float*>(nullptr));
  });
}

// The same where b is a's type or float.
template <class F>
void with_param_types(int a, int b, F&& f) {
  with_type(a, [&](auto* pa) {
    if (a == b) f(pa, pa);
    else if constexpr (!std::is_same_v<decltype(pa), float*>) f(pa, static_cast<float*>(nullptr));
  });
}

// Calls f with the widest VE that the two matrices' rows allow: 16 bytes of
// T, four or two 16-bit values, or one value.
template <class T, class F>
void with_width(const Mat& a, uint64_t a_rows, const Mat& b, uint64_t b_rows, uint64_t dim, F&& f) {
  const auto fits = [&](uint64_t n) {
    return dim % n == 0 && row_aligned(a.data, a.stride, a_rows, type_size(a.type), n) &&
           row_aligned(b.data, b.stride, b_rows, type_size(b.type), n);
  };
  constexpr int kWide = 16 / sizeof(T);
  if (fits(kWide)) return f(std::integral_constant<int, kWide>());
  if constexpr (kWide > 4) {
    if (fits(4)) return f(std::integral_constant<int, 4>());
    if (fits(2)) return f(std::integral_constant<int, 2>());
  }
  f(std::integral_constant<int, 1>());
}

}  // namespace xgbb::nn
