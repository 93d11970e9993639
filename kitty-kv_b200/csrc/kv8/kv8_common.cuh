// Shared pieces of the 8-bit cache kernels: the host-side checks, the sticky device
// error bits and the conversions between 16-bit rows, 8-bit codes and float32.
//
// Times in these files are of calls replayed from a CUDA graph in a burst on one B200 at full
// clocks, over three caches, unless they say otherwise.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <cstdio>
#include <cstring>

#include "../../../include/kitty_b200.h"
#include "../../../include/kitty_kv8.h"

namespace kitty8 {

constexpr uint32_t kErrPage = 1u << 1, kErrRows = 1u << 2, kErrSlot = 1u << 3, kErrLength = 1u << 4,
                   kErrPosition = 1u << 5;

// The message is kept in a fixed thread-local buffer, so that no entry point can throw.
int fail(int code, const char* what, const char* msg);
int check_launch(const char* what);
int sm_count();                       // of the current device
uint32_t* error_word();               // device address of the sticky bits on the current device (host call)
int check_cache(const KittyKv8Cache* c, const char* what);

// Launch as a programmatic dependent of whatever is before it on the stream: the launch itself
// overlaps the end of that, and the kernel waits (dev::wait_for_stream, before it touches
// memory) until it is done.  Between the short kernels of a decode step that is 1 to 2 us:
// eager calls of 256 single-token writes 6.1 -> 4.6 us, of a read of 4137 tokens 8.2 -> 6.5, of
// attention over 4133 tokens 14.3 -> 12.4.
template <typename... Params, typename... Args>
int launch_dependent(const char* what, void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t s,
                     Args... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
  if (e == cudaSuccess) return KITTY_OK;
  cudaGetLastError();                  // reported here, and not to whoever asks next
  return fail(KITTY_ERR_CUDA, what, cudaGetErrorString(e));
}

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

namespace dev {

// What was before this kernel on its stream is done, and its writes are visible (to loads that
// are not marked read-only).
__device__ __forceinline__ void wait_for_stream() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ void flag(uint32_t* word, uint32_t bits) { atomicOr(word, bits); }

template <bool kBf16>
__device__ __forceinline__ float2 to_f2(uint32_t x) {
  if constexpr (kBf16) {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  } else {
    __half2 h;
    memcpy(&h, &x, 4);
    return __half22float2(h);
  }
}

template <bool kBf16>
__device__ __forceinline__ uint32_t from_f2(float lo, float hi) {
  uint32_t r;
  if constexpr (kBf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// |x| of a packed pair, and the NaN-propagating maximum of two packed pairs.
__device__ __forceinline__ uint32_t abs2(uint32_t x) { return x & 0x7fff7fffu; }
template <bool kBf16>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (kBf16)
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// 8-bit codes of four values (first value in the lowest byte): round to nearest even,
// saturating; NaN gives e4m3 NaN or int8 0.
template <int kCode>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if constexpr (kCode == KITTY_KV8_E4M3) {
    uint32_t lo, hi;
    asm("{\n .reg .b16 t;\n cvt.rn.satfinite.e4m3x2.f32 t, %1, %2;\n cvt.u32.u16 %0, t;\n}"
        : "=r"(lo) : "f"(b), "f"(a));
    asm("{\n .reg .b16 t;\n cvt.rn.satfinite.e4m3x2.f32 t, %1, %2;\n cvt.u32.u16 %0, t;\n}"
        : "=r"(hi) : "f"(d), "f"(c));
    return lo | (hi << 16);
  } else {
    auto one = [](float x) -> uint32_t {   // the conversion saturates to 32 bits and takes NaN to 0
      return static_cast<uint32_t>(max(-127, min(127, __float2int_rn(x)))) & 0xffu;
    };
    return one(a) | (one(b) << 8) | (one(c) << 16) | (one(d) << 24);
  }
}

// float32 values of the four codes of a word.
template <int kCode>
__device__ __forceinline__ float4 decode4(uint32_t w) {
  if constexpr (kCode == KITTY_KV8_E4M3) {
    uint32_t lo, hi;
    asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
        : "=r"(lo), "=r"(hi) : "r"(w));
    const float2 x = to_f2<false>(lo), y = to_f2<false>(hi);
    return make_float4(x.x, x.y, y.x, y.y);
  } else {
    return make_float4(float(int8_t(w)), float(int8_t(w >> 8)), float(int8_t(w >> 16)), float(int8_t(w >> 24)));
  }
}

// Number of the n values of the ascending array a that are <= v, by the whole warp: each
// step looks at 32 evenly spaced values at once.  Any contents end within the bounds.
__device__ __forceinline__ int count_le(const int32_t* a, int n, int v) {
  const int lane = threadIdx.x & 31;
  int lo = 0, len = n;                 // the answer lies in [lo, lo + len]
  while (len > 0) {
    const int step = (len + 31) / 32;
    const int at = lo + lane * step;   // the last value of each part but the last is not looked at
    const bool le = at < lo + len && a[at] <= v;
    const int k = __popc(__ballot_sync(0xffffffffu, le));
    if (k == 0) return lo;
    const int next = lo + (k - 1) * step + 1;
    len = min(step - 1, lo + len - next);
    lo = next;
  }
  return lo;
}

// Whether entry i's slot is given by an earlier entry too (by the whole warp).
__device__ __forceinline__ bool repeated(const int32_t* seq_map, int i, int slot) {
  bool hit = false;
  for (int j = threadIdx.x & 31; j < i; j += 32) hit |= seq_map[j] == slot;
  return __any_sync(0xffffffffu, hit);
}

}  // namespace dev
}  // namespace kitty8
