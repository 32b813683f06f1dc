// Eight neighbouring elements of a row as 32-bit floats, and the microscaled formats: blocks of 32 that share a power of two.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tc_kernels.cuh"

namespace tck {

// ---- eight elements of a type ----
template <class T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int kWords = 8;  // 32-bit words of eight elements
  static constexpr float kMost = 3.402823466e38f;
  __device__ __forceinline__ static float get(float v) { return v; }
  __device__ __forceinline__ static float put(float v) { return v; }
  __device__ __forceinline__ static void unpack(const uint32_t* w, float* f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
  }
  __device__ __forceinline__ static void pack(const float* f, uint32_t* w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(f[i]);
  }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kWords = 4;
  static constexpr float kMost = 3.3895313892515355e38f;
  __device__ __forceinline__ static float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ __forceinline__ static __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
  __device__ __forceinline__ static void unpack(const uint32_t* w, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
  }
  __device__ __forceinline__ static void pack(const float* f, uint32_t* w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("cvt.rn.bf16x2.f32 %0, %2, %1;\n" : "=r"(w[i]) : "f"(f[2 * i]), "f"(f[2 * i + 1]));
  }
};
template <>
struct Elem<__half> {
  static constexpr int kWords = 4;
  static constexpr float kMost = 65504.f;
  __device__ __forceinline__ static float get(__half v) { return __half2float(v); }
  __device__ __forceinline__ static __half put(float v) { return __float2half_rn(v); }
  __device__ __forceinline__ static void unpack(const uint32_t* w, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(w + i));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
  __device__ __forceinline__ static void pack(const float* f, uint32_t* w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("cvt.rn.f16x2.f32 %0, %2, %1;\n" : "=r"(w[i]) : "f"(f[2 * i]), "f"(f[2 * i + 1]));
  }
};

// Eight elements of a row as they lie in memory.  Vec: their address and the row's end allow 16-byte accesses; else one by one,
// those from `valid` on zeros (loads) or left alone (stores).
template <class T>
struct Raw {
  uint32_t w[Elem<T>::kWords];
};
template <class T, bool Vec>
__device__ __forceinline__ Raw<T> load8(const T* p, int valid) {
  Raw<T> r;
  if constexpr (Vec) {
#pragma unroll
    for (int i = 0; i < Elem<T>::kWords; i += 4) {
      const uint4 v = valid > 0 ? *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i) : make_uint4(0, 0, 0, 0);
      r.w[i] = v.x; r.w[i + 1] = v.y; r.w[i + 2] = v.z; r.w[i + 3] = v.w;
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = i < valid ? reinterpret_cast<const uint32_t*>(p)[i] : 0u;
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = (2 * i < valid ? (uint32_t)q[2 * i] : 0u) | (2 * i + 1 < valid ? (uint32_t)q[2 * i + 1] << 16 : 0u);
  }
  return r;
}
template <class T, bool Vec>
__device__ __forceinline__ void store8(T* p, const Raw<T>& r, int valid) {
  if constexpr (Vec) {
    if (valid > 0) {
#pragma unroll
      for (int i = 0; i < Elem<T>::kWords; i += 4)
        *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(p) + i) = make_uint4(r.w[i], r.w[i + 1], r.w[i + 2], r.w[i + 3]);
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) reinterpret_cast<uint32_t*>(p)[i] = r.w[i];
  } else {
    uint16_t* q = reinterpret_cast<uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) q[i] = (uint16_t)(r.w[i >> 1] >> (16 * (i & 1)));
  }
}
template <class T>
__device__ __forceinline__ void unpack8(const Raw<T>& r, float* f) { Elem<T>::unpack(r.w, f); }
template <class T>
__device__ __forceinline__ Raw<T> pack8(const float* f) {
  Raw<T> r;
  Elem<T>::pack(f, r.w);
  return r;
}

// ---- two floats at a time ----
typedef unsigned long long F2;
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 f2(float a) { return f2(a, a); }
__device__ __forceinline__ float2 of2(F2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ float sum2(F2 v) {
  const float2 r = of2(v);
  return r.x + r.y;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
template <class T>
__device__ __forceinline__ void unpack8(const Raw<T>& r, F2 (&v)[4]) {
  float f[8];
  Elem<T>::unpack(r.w, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = f2(f[2 * i], f[2 * i + 1]);
}
template <class T>
__device__ __forceinline__ Raw<T> pack8(const F2 (&v)[4]) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = of2(v[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
  return pack8<T>(f);
}

// ---- microscaled blocks ----
// A block's scale 2^e as the byte e + 127: the smallest (from 0 on) for which the largest magnitude, given by its bits, is at most
// L * 2^e; 255 where there is an infinity or a NaN.  L = 6 = 1.5 * 2^2 (e2m1) or 448 = 1.75 * 2^8 (e4m3): exponents are compared as
// whole numbers and the mantissa with L's, so nothing is rounded.
__device__ __forceinline__ uint32_t micro4_scale(uint32_t amax) {
  return amax >= 0x7F800000u ? 255u : (uint32_t)max((int)(amax >> 23) - 2 + ((amax & 0x7FFFFFu) > 0x400000u ? 1 : 0), 0);
}
__device__ __forceinline__ uint32_t micro8_scale(uint32_t amax) {
  return amax >= 0x7F800000u ? 255u : (uint32_t)max((int)(amax >> 23) - 8 + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0), 0);
}
// 2^(byte - 127); NaN for 255.
__device__ __forceinline__ float micro_power(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7FFFFFFFu) : byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
// 2^(127 - byte), by which a finite value of the block is scaled without rounding down to where its code is zero anyway.
__device__ __forceinline__ float micro_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// The largest magnitude of a lane's eight elements, as the bits of a float: 16-bit types two at a time, their bits order as numbers do.
template <class T>
__device__ __forceinline__ uint32_t magnitude_of(const Raw<T>& r) {
  if constexpr (sizeof(T) == 4) {
    return max(max(max(r.w[0] & 0x7FFFFFFFu, r.w[1] & 0x7FFFFFFFu), max(r.w[2] & 0x7FFFFFFFu, r.w[3] & 0x7FFFFFFFu)),
               max(max(r.w[4] & 0x7FFFFFFFu, r.w[5] & 0x7FFFFFFFu), max(r.w[6] & 0x7FFFFFFFu, r.w[7] & 0x7FFFFFFFu)));
  } else {
    uint32_t m = __vmaxu2(__vmaxu2(r.w[0] & 0x7FFF7FFFu, r.w[1] & 0x7FFF7FFFu), __vmaxu2(r.w[2] & 0x7FFF7FFFu, r.w[3] & 0x7FFF7FFFu));
    m = max(m >> 16, m & 0xFFFFu);
    const uint16_t h = (uint16_t)m;
    return __float_as_uint(Elem<T>::get(*reinterpret_cast<const T*>(&h)));
  }
}
// Over the four neighbouring lanes that hold a block.
__device__ __forceinline__ uint32_t block_max(uint32_t m) {
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
}

// Eight scaled values to e2m1, two a byte, the first in the low half: to nearest, ties to even.
__device__ __forceinline__ uint32_t to_e2m1(const float* f) {
  uint32_t r;
  asm("{\n .reg .b8 a, b, c, d;\n"
      " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      " mov.b32 %0, {a, b, c, d};\n}\n"
      : "=r"(r)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return r;
}
__device__ __forceinline__ void from_e2m1(uint32_t code, float* f) {
  uint32_t h[4];
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n"
      " cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}\n"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(code));
  Elem<__half>::unpack(h, f);
}
// Eight scaled values to e4m3, the first in the lowest byte: to nearest, ties to even.
__device__ __forceinline__ uint2 to_e4m3(const float* f) {
  uint16_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;\n" : "=h"(h[i]) : "f"(f[2 * i]), "f"(f[2 * i + 1]));
  return make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
}
__device__ __forceinline__ void from_e4m3(uint2 code, float* f) {
  uint32_t h[4];
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h[0]) : "h"((uint16_t)code.x));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h[1]) : "h"((uint16_t)(code.x >> 16)));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h[2]) : "h"((uint16_t)code.y));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h[3]) : "h"((uint16_t)(code.y >> 16)));
  Elem<__half>::unpack(h, f);
}
// Values of a block; what rounding took past the type's largest number is that number.  Only the largest scales reach there.
template <class T>
__device__ __forceinline__ void rescale8(float* f, uint32_t byte) {
  const float scale = micro_power(byte);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] *= scale;
  constexpr uint32_t kFar = sizeof(T) == 2 && Elem<T>::kMost < 1e5f ? 127 + 15 - 8 : 127 + 127 - 8;  // 2^e times 2^8 may pass it
  if (byte >= kFar) {
    constexpr float most = Elem<T>::kMost;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = f[i] > most ? most : f[i] < -most ? -most : f[i];  // NaN stays
  }
}

// ---- rows in units of 128 columns: 16 lanes, eight columns each ----
// Where 16-byte accesses do not reach, a unit goes through `stage` (shared memory, 128 elements of the lanes' own), so that
// neighbouring lanes touch neighbouring elements.  All lanes of the warp call these.
template <class T, bool Vec>
__device__ __forceinline__ Raw<T> unit_load(const T* unit, int lane, int valid, T* stage) {  // valid: columns from the unit's first to the row's end
  if constexpr (Vec) {
    return load8<T, true>(unit + lane * 8, valid - lane * 8);
  } else {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = i * 16 + lane;
      stage[c] = c < valid ? unit[c] : Elem<T>::put(0.f);
    }
    __syncwarp();
    return load8<T, true>(stage + lane * 8, 8);
  }
}
template <class T, bool Vec>
__device__ __forceinline__ void unit_store(T* unit, const Raw<T>& r, int lane, int valid, T* stage) {
  if constexpr (Vec) {
    store8<T, true>(unit + lane * 8, r, valid - lane * 8);
  } else {
    __syncwarp();
    store8<T, true>(stage + lane * 8, r, 8);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = i * 16 + lane;
      if (c < valid) unit[c] = stage[c];
    }
  }
}

}  // namespace tck

// Whether 16-byte accesses reach every group of eight elements of rows of `cols` elements.
inline bool tc_vec8(const void* p, int64_t ld, int64_t cols, int es) {
  return !(reinterpret_cast<uintptr_t>(p) & 15) && (ld * es) % 16 == 0 && cols % 8 == 0;
}
inline bool tc_odd_address(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }
