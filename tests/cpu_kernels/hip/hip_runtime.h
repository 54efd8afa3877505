// Stands for HIP's header when the token operators' kernels are compiled for the CPU
// (tests/test_token_ops_cpu.py): a block's threads are fibers (block.cpp), what 64 of
// them do together is an exchange between their slots, and shared memory is static.  Only
// what those kernels use is here.
#pragma once
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <functional>

#define __device__
#define __host__
#define __global__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __restrict__
#define __shared__ static

struct float2 { float x, y; };
struct alignas(16) float4 { float x, y, z, w; };
inline float2 make_float2(float a, float b) { return {a, b}; }
inline float4 make_float4(float a, float b, float c, float d) { return {a, b, c, d}; }
struct dim3 {
  unsigned x, y, z;
  dim3(unsigned a = 1, unsigned b = 1, unsigned c = 1) : x(a), y(b), z(c) {}
};
struct Index { unsigned x, y, z; };
typedef void* hipStream_t;

extern Index threadIdx, blockIdx, gridDim, blockDim;
extern char* dynamic_lds;
// every live lane of the wave gives v and gets all of them, and which lanes are live
void wave_exchange(uint64_t v, uint64_t* all, uint64_t* live);
void block_barrier();
void run_grid(dim3 grid, dim3 block, size_t lds, const std::function<void()>& kernel, const char* name);

inline int64_t grid_threads() {
  const char* e = getenv("GRID_THREADS");
  return e ? atoll(e) : (int64_t(1) << 32) - 1;
}

#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) \
  run_grid(grid, block, lds, [=]() { kernel(__VA_ARGS__); }, #kernel)
#define __syncthreads() block_barrier()

template <typename To, typename From>
To bits_as(From v) {
  static_assert(sizeof(To) == sizeof(From), "size");
  To o;
  memcpy(&o, &v, sizeof o);
  return o;
}
inline uint32_t __float_as_uint(float f) { return bits_as<uint32_t>(f); }
inline int __float_as_int(float f) { return bits_as<int>(f); }
inline float __uint_as_float(uint32_t u) { return bits_as<float>(u); }
inline float __int_as_float(int u) { return bits_as<float>(u); }
inline int __popcll(uint64_t v) { return __builtin_popcountll(v); }

struct Lanes {  // what every lane gave
  uint64_t v[64], live;
  template <typename T>
  explicit Lanes(T mine) {
    uint64_t u = 0;
    memcpy(&u, &mine, sizeof mine);
    wave_exchange(u, v, &live);
  }
  template <typename T>
  T at(int lane) const {
    T o;
    memcpy(&o, &v[lane], sizeof o);
    return o;
  }
};
inline int lane_id() { return threadIdx.x & 63; }
inline uint64_t __ballot(int p) {
  const Lanes a(p != 0 ? 1 : 0);
  uint64_t m = 0;
  for (int i = 0; i < 64; ++i)
    if ((a.live >> i) & 1 && a.at<int>(i)) m |= uint64_t(1) << i;
  return m;
}
template <typename T>
T __shfl_xor(T v, int o, int) { return Lanes(v).template at<T>(lane_id() ^ o); }
template <typename T>
T __shfl_up(T v, int o, int) {
  const Lanes a(v);
  return lane_id() >= o ? a.at<T>(lane_id() - o) : v;
}
inline int __builtin_amdgcn_update_dpp(int, int v, int ctrl, int, int, bool) {
  const Lanes a(v);
  const int l = lane_id();
  if (ctrl < 0x100) return a.at<int>((l & ~3) | ((ctrl >> (2 * (l & 3))) & 3));  // quad_perm
  if (ctrl == 0x140) return a.at<int>((l & ~15) | (15 - (l & 15)));               // row_mirror
  if (ctrl == 0x141) return a.at<int>((l & ~7) | (7 - (l & 7)));                  // row_half_mirror
  abort();
}
struct LanePair { uint32_t v[2]; uint32_t operator[](int i) const { return v[i]; } };
inline LanePair lane_pair(uint32_t mine, int bit) {
  const Lanes a(mine);
  return {{a.at<uint32_t>(lane_id() & ~bit), a.at<uint32_t>(lane_id() | bit)}};
}
#define __builtin_amdgcn_permlane16_swap(a, b, c, d) lane_pair(a, 16)
#define __builtin_amdgcn_permlane32_swap(a, b, c, d) lane_pair(a, 32)
#define __builtin_amdgcn_exp2f exp2f
#define __builtin_amdgcn_fence(...) ((void)0)
#define __builtin_amdgcn_wave_barrier() ((void)Lanes(0))
#define __HIP_MEMORY_SCOPE_WORKGROUP 0
#define __hip_atomic_store(p, v, order, scope) (*(p) = (v))
#define __hip_atomic_load(p, order, scope) (*(p))
template <typename T>
T atomicAdd(T* p, T v) {
  const T old = *p;
  *p += v;
  return old;
}
