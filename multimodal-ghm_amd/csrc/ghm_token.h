// Shared by the token operators (ghm_score.hip, ghm_distill.hip, ghm_embed.hip): value
// types, token ids, 16-byte vectors at any alignment, wave and group reductions, and the
// one-pass scan of a logits row.
//
// Logits rows are addressed as base + (r / n_inner) * s_outer + (r % n_inner) * s_inner
// elements, so a view past leading positions ([N][T][V] from position P on) is read
// in place.  Values are f32, bf16 or f16; every sum, maximum and statistic is f32.
#pragma once
#include "ghm_common.h"
#include "ghm_launch.h"

#include <float.h>
#include <type_traits>

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float NEG_INF = -__builtin_inff();

struct bf16_t { uint16_t u; };
struct f16_t { _Float16 h; };

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(bf16_t x) { return __uint_as_float(static_cast<uint32_t>(x.u) << 16); }
__device__ __forceinline__ float to_f(f16_t x) { return static_cast<float>(x.h); }
__device__ __forceinline__ void from_f(float& o, float x) { o = x; }
__device__ __forceinline__ void from_f(bf16_t& o, float x) { o.u = __builtin_bit_cast(uint16_t, static_cast<__bf16>(x)); }
__device__ __forceinline__ void from_f(f16_t& o, float x) { o.h = static_cast<_Float16>(x); }

struct Rows {
  const void* base;
  int64_t n_inner, s_outer, s_inner;
};
template <typename T>
__device__ __forceinline__ const T* row_ptr(const Rows& m, int64_t r) {
  return static_cast<const T*>(m.base) + (r / m.n_inner) * m.s_outer + (r % m.n_inner) * m.s_inner;
}

// token ids of 8 (unsigned), 32 or 64 bits
struct Ids {
  const void* p;
  int bits;
};
__device__ __forceinline__ int64_t ld_id(const Ids& t, int64_t i) {
  if (t.bits == 64) return static_cast<const int64_t*>(t.p)[i];
  if (t.bits == 32) return static_cast<const int32_t*>(t.p)[i];
  return static_cast<const uint8_t*>(t.p)[i];
}

// several at once: no load waits for another's branch
template <int U, typename F>
__device__ __forceinline__ void ld_ids(const Ids& t, int64_t (&id)[U], F at) {
  if (t.bits == 64) {
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = static_cast<const int64_t*>(t.p)[at(u)];
  } else if (t.bits == 32) {
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = static_cast<const int32_t*>(t.p)[at(u)];
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = static_cast<const uint8_t*>(t.p)[at(u)];
  }
}

// Order of the alternatives: value descending (NaN above all, -0 equal to +0),
// then id ascending, as one unsigned 64-bit key per entry.
__device__ __forceinline__ uint32_t order_bits(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (static_cast<int32_t>(u) < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint64_t top_key(float x, uint32_t id) {
  return (static_cast<uint64_t>(order_bits(x)) << 32) | (0xffffffffu - id);
}

// 16 bytes of a row as floats, and back, at any element alignment
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
template <typename T>
struct Vec {
  static constexpr int N = 8;
  using raw = u32x4_a2;
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  using raw = u32x4_a4;
};
template <typename T, int N>
__device__ __forceinline__ void unpack(u32x4 v, float (&x)[N]) {
  static_assert(N == Vec<T>::N, "16 bytes");
  T e[N];
  __builtin_memcpy(e, &v, 16);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = to_f(e[i]);
}
template <int N, typename T>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[N]) {
  if constexpr (N == 1) x[0] = to_f(*p);
  else unpack<T>(*reinterpret_cast<const typename Vec<T>::raw*>(p), x);
}
// STREAM: past the caches (worth it for whole lines that nothing reads again soon)
template <int N, bool STREAM = false, typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[N]) {
  if constexpr (N == 1) {
    from_f(*p, x[0]);
  } else {
    T e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) from_f(e[i], x[i]);
    u32x4 v;
    __builtin_memcpy(&v, e, 16);
    if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<typename Vec<T>::raw*>(p));
    else *reinterpret_cast<typename Vec<T>::raw*>(p) = v;
  }
}

// the block's number in a grid of grid_of
__device__ __forceinline__ int64_t block_number() { return static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x; }

// f over the 64 lanes, in every lane, on the vector unit alone: lane pairs, quads, eights and
// rows of 16 by DPP, then rows 0 / 1 and 2 / 3, then the halves.  (Through the LDS crossbar
// a distillation step of 111,848 rows of 600 values, seven of these each, took 238 us.)
template <typename F>
__device__ __forceinline__ float wave_all(float v, F f) {
  const auto dpp = [](float x, auto ctrl) {
    const int i = __float_as_int(x);
    return __int_as_float(__builtin_amdgcn_update_dpp(i, i, decltype(ctrl)::value, 0xf, 0xf, false));
  };
  v = f(v, dpp(v, std::integral_constant<int, 0xb1>()));   // quad_perm 1 0 3 2
  v = f(v, dpp(v, std::integral_constant<int, 0x4e>()));   // quad_perm 2 3 0 1
  v = f(v, dpp(v, std::integral_constant<int, 0x141>()));  // row_half_mirror
  v = f(v, dpp(v, std::integral_constant<int, 0x140>()));  // row_mirror
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ float wave_max(float v) {
  return wave_all(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_all(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ void wave_fence() {  // this wave's LDS writes before its later reads
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A group of W waves works on one row (W == 1: no barrier, the block holds several).
// Reductions go through slots of LDS in a fixed order; every use names a slot of its own.
template <int W>
__device__ __forceinline__ void group_sync() {
  if constexpr (W > 1) __syncthreads();
  else wave_fence();
}
template <int W>
__device__ __forceinline__ float group_max(float v, float* slot, int w) {
  v = wave_max(v);
  if constexpr (W == 1) return v;
  if ((threadIdx.x & 63) == 0) slot[w] = v;
  __syncthreads();
  v = slot[0];
#pragma unroll
  for (int i = 1; i < W; ++i) v = fmaxf(v, slot[i]);
  return v;
}
template <int W>
__device__ __forceinline__ float group_sum(float v, float* slot, int w) {
  v = wave_sum(v);
  if constexpr (W == 1) return v;
  if ((threadIdx.x & 63) == 0) slot[w] = v;
  __syncthreads();
  v = slot[0];
#pragma unroll
  for (int i = 1; i < W; ++i) v += slot[i];
  return v;
}

// One pass over a row: a lane's running maximum m and sums relative to it.
//   s = sum e^{c1 (z - m)};  SECOND_ENT: t = sum e^{c1 d} d (d = z - m);
//   SECOND_EXP: t = sum e^{c2 d};  SECOND_NONE: t unused.
// The maximum starts at the lowest finite value, so differences never are -inf minus
// -inf; where a difference is a factor of the entropy's sum it is cut at -1e4 (e^-1e4 = 0, and
// 0 times -inf is not).  An exponent's difference is never cut: c1 and c2 carry log2 e over a
// temperature of up to 10^6, where e^(-1e4 / 10^6) is 0.99.  NaN and +inf make s NaN.
// EXACT: values at the maximum are counted in n and not added to the sums, so that the
// logarithm of a sum just above 1 keeps its digits (log1p): a row with one likely value
// of few.  Rows of up to 256 values afford the two instructions per value.
enum { SECOND_NONE, SECOND_ENT, SECOND_EXP };
struct Sums {
  float m = -FLT_MAX, s = 0.f, t = 0.f, n = 0.f;
  __device__ __forceinline__ float total() const { return n + s; }
  __device__ __forceinline__ float log_s() const { return n == 1.f ? log1pf(s) : logf(n + s); }
  __device__ __forceinline__ float log_t() const { return n == 1.f ? log1pf(t) : logf(n + t); }  // SECOND_EXP
};
template <int SECOND>
__device__ __forceinline__ void rebase(Sums& a, float m, float c1, float c2) {
  const float dm = a.m - m, f = __builtin_amdgcn_exp2f(dm * c1);
  const float n = dm == 0.f ? 0.f : a.n;  // what was at the old maximum joins the sums
  if constexpr (SECOND == SECOND_ENT) a.t = f * (a.t + fmaxf(dm, -1e4f) * (a.s + n));
  if constexpr (SECOND == SECOND_EXP) a.t = __builtin_amdgcn_exp2f(dm * c2) * (a.t + n);
  a.s = f * (a.s + n);
  a.n -= n;
  a.m = m;
}
template <int SECOND, bool EXACT, int N>
__device__ __forceinline__ void fold(Sums& a, const float (&x)[N], float c1, float c2) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = x[i] - a.m, e = __builtin_amdgcn_exp2f(d * c1);
    const bool top = EXACT && d == 0.f;
    if constexpr (EXACT) a.n += top ? 1.f : 0.f;
    a.s += top ? 0.f : e;
    if constexpr (SECOND == SECOND_ENT) a.t += e * fmaxf(d, -1e4f);
    if constexpr (SECOND == SECOND_EXP) a.t += top ? 0.f : __builtin_amdgcn_exp2f(d * c2);
  }
}
// the group's sums in every lane
template <int SECOND, int W>
__device__ __forceinline__ Sums group_join(Sums a, float* slots, int w, float c1, float c2) {
  rebase<SECOND>(a, group_max<W>(a.m, slots, w), c1, c2);
  a.s = wave_sum(a.s);
  if constexpr (SECOND != SECOND_NONE) a.t = wave_sum(a.t);
  if constexpr (W == 1) a.n = wave_sum(a.n);  // EXACT rows are one wave's
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) {
      slots[W + w] = a.s;
      if constexpr (SECOND != SECOND_NONE) slots[2 * W + w] = a.t;
    }
    __syncthreads();
    a.s = slots[W];
#pragma unroll
    for (int i = 1; i < W; ++i) a.s += slots[W + i];
    if constexpr (SECOND != SECOND_NONE) {
      a.t = slots[2 * W];
#pragma unroll
      for (int i = 1; i < W; ++i) a.t += slots[2 * W + i];
    }
  }
  return a;
}

// ---- the largest values of a row, found in the same pass -------------------
// The unit kept is a lane's vector of N values, by its maximum (value descending, index
// ascending, as a 64-bit key): the k largest values lie in the k largest vectors, since
// each of k vectors ranked above another holds a value that ranks above all of that one's.
// A wave notes in LDS the vectors above a threshold that only rises.  Valid thresholds:
// (a) with r = ceil(k / W), the least over the waves of each wave's r-th largest lane
// maximum: the waves hold k vectors at or above it; (b) a wave's own k-th vector after a
// prune, strictly, for its later (higher) indices.  That is one comparison per vector, and
// a few hundred vectors of a row are noted; at the end they are ranked by counting, and
// the values of the k best ones, read again, are ranked the same way.  The maxima skip NaN:
// a range whose sum is NaN (a NaN or +inf in it) is searched value by value instead.
constexpr int TOP_CAP = 384;  // vectors noted per wave: pruned where a batch might not fit
constexpr int TOP_BATCH = 256;  // vectors of a wave's batch, at most

// at least r lanes hold u >= the result (its upper 16 bits are searched: a lower bound
// of the r-th largest); 0: fewer
__device__ __forceinline__ uint32_t kth_bits(uint32_t u, int r) {
  uint32_t K = 0;
#pragma unroll
  for (int b = 31; b >= 16; --b) {
    const uint32_t c = K | (1u << b);
    if (__popcll(__ballot(u >= c)) >= r) K = c;
  }
  return K;
}
// the float just below order bits K: x > it is order_bits(x) >= K.  NaN (nothing is at
// or below it) if K is no more than what a lane without values holds.
__device__ __forceinline__ float below(uint32_t K) {
  if (K <= 0x00800000u) return __builtin_nanf("");
  const uint32_t o = K - (K == 0x80000000u ? 2 : 1);  // -0 is equal to +0, not below it
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}

// keep the k largest of a wave's n candidates, in descending order (spare: 64 words)
__device__ __forceinline__ void top_prune(uint64_t* cand, uint64_t* spare, int n, int k, int lane) {
  wave_fence();
#pragma unroll 1
  for (int j = lane; j < n; j += 64) {
    const uint64_t mine = cand[j];
    int rank = 0;
#pragma unroll 1
    for (int i = 0; i < n; ++i) rank += cand[i] > mine;
    if (rank < k) spare[rank] = mine;
  }
  wave_fence();
  if (lane < k) cand[lane] = spare[lane];
  wave_fence();
}

// What finding the alternatives takes in LDS per group of W waves.
template <int N, int W>
struct TopLds {
  uint64_t cand[W * TOP_CAP], merged[W * 64], best[N == 1 ? 1 : GHM_TOP_MAX], vals[N == 1 ? 1 : GHM_TOP_MAX * N];
  uint32_t bound[W];
  int count[W], n_vals;
};
struct TopState {
  int cnt = 0;         // vectors this wave has noted
  uint32_t bound = 0;  // the group's bound (a) as order bits
};

// A row's values lo .. hi - 1 (of at least N in the row up to hi): batches of U vectors of N
// values per lane; the values after the last whole vector are one more vector, read as the
// range's last N values with those that the vector before holds masked.  The vectors of
// a wave come in ascending order.  TOP: notes vectors for the k largest values.
template <typename T, int N, int U, int W, int SECOND, bool TOP>
__device__ __forceinline__ Sums scan_row(const T* z, int lo, int hi, float c1, float c2, int w, int lane, int k,
                                         TopLds<N, W>* lds, TopState& top) {
  Sums a;
  float thr = __builtin_nanf("");
  const int tail = (hi - lo) % N, nv = (hi - lo) / N + (tail ? 1 : 0);
  const int r = TOP ? (k + W - 1) / W : 0;
  constexpr int STEP = W * 64 * U;
  const int nb = (nv + STEP - 1) / STEP;
  uint64_t* cand = TOP ? lds->cand + w * TOP_CAP : nullptr;
  for (int b = 0; b < nb; ++b) {
    float x[U][N], vm[U];
    const int v0 = b * STEP + w * 64 + lane;
    if (b < nb - 1) {
#pragma unroll
      for (int u = 0; u < U; ++u) load_vec<N>(z + lo + (v0 + u * W * 64) * N, x[u]);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {  // lanes past the end read the last vector again
        const int v = v0 + u * W * 64, at = v < nv ? v * N : (nv - 1) * N;
        load_vec<N>(z + (lo + at + N <= hi ? lo + at : hi - N), x[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int v = v0 + u * W * 64;
        const int skip = v >= nv ? N : v == nv - 1 && tail ? N - tail : 0;
#pragma unroll
        for (int i = 0; i < N; ++i) x[u][i] = i < skip ? NEG_INF : x[u][i];
      }
    }
    float bm = -FLT_MAX;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      vm[u] = x[u][0];
#pragma unroll
      for (int i = 1; i < N; ++i) vm[u] = fmaxf(vm[u], x[u][i]);
      bm = fmaxf(bm, vm[u]);
    }
    rebase<SECOND>(a, fmaxf(a.m, bm), c1, c2);
#pragma unroll
    for (int u = 0; u < U; ++u) fold<SECOND, N == 1>(a, x[u], c1, c2);
    if constexpr (TOP) {
      if (((b + 1) & b) == 0 || b == nb - 1) {  // the shared bound, after batches 1, 2, 4, 8, ... and the last
        const uint32_t K = kth_bits(order_bits(a.m), r);
        top.bound = K;
        if constexpr (W > 1) {
          if (lane == 0) __hip_atomic_store(lds->bound + w, K, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
          if (b == 0) __syncthreads();
#pragma unroll
          for (int i = 0; i < W; ++i) {
            const uint32_t o = __hip_atomic_load(lds->bound + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            top.bound = o < top.bound ? o : top.bound;
          }
        }
        thr = fmaxf(thr, below(top.bound));  // fmaxf takes the other of a NaN
      }
      if (__ballot(!(bm <= thr)) == 0) continue;
      static_assert(64 * U <= TOP_BATCH, "a batch fits beside what a prune leaves");
      if (top.cnt > TOP_CAP - TOP_BATCH) {
        top_prune(cand, lds->merged + w * 64, top.cnt, k, lane);
        top.cnt = k;
        thr = fmaxf(thr, key_value(cand[k - 1]));
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int v = v0 + u * W * 64;
        const uint64_t mask = __ballot(v < nv && !(vm[u] <= thr));
        if ((mask >> lane) & 1) cand[top.cnt + __popcll(mask & ((uint64_t(1) << lane) - 1))] = top_key(vm[u], v);
        top.cnt += __popcll(mask);
      }
    }
  }
  return a;
}

constexpr int SHORT_V = 32;  // rows of at most this many values: one lane per row

// Rows of up to 256 vectors take one wave, up to 1,536 too where there are many of them
// (scores of 16,777 rows of 4,000 bf16 values: 30 us by one wave, 34 by two, 56 by four).
inline bool one_wave(int64_t rows, int64_t V, int N) {
  return V <= 256 * N || (V <= 1536 * N && rows >= 1024);
}

// Few, long rows go in parts of at least 4,096 values, about 512 in all, and a second launch
// joins a row's parts: only where that pays for the launch (4 rows of 131,072 bf16 values
// with 20 alternatives: 12 us in parts, 18 whole; of 32,000 values: 11 and 9.5).  The
// callers' thresholds, in vectors and rows:
constexpr int MAX_PARTS = 64;  // of a row
struct Split {
  int parts, len;
};
struct SplitRule {
  int64_t vectors, rows;
};
constexpr SplitRule SPLIT_TOP{8192, 511};   // scores with alternatives
constexpr SplitRule SPLIT_SUMS{32768, 64};  // sums alone: 100 rows of 131,072 f32 values 15 us in parts, 14 whole
constexpr SplitRule SPLIT_STEP{16384, 32};  // sums and gradient: 100 rows of 131,072 bf16 values 33 us in parts, 26 whole
inline Split row_split(int64_t rows, int64_t V, int N, SplitRule rule) {
  if (rows < 1 || rows > rule.rows || V <= rule.vectors * N) return {1, static_cast<int>(V)};
  int64_t p = (512 + rows - 1) / rows;
  if (p > V / 4096) p = V / 4096;
  if (p > MAX_PARTS) p = MAX_PARTS;
  int64_t len = (V + p - 1) / p;
  len = (len + 511) / 512 * 512;
  return {static_cast<int>((V + len - 1) / len), static_cast<int>(len)};
}

// f(value) over a row's values lo .. hi - 1, written to d in batches of U vectors.  LINES: from
// d's first 64-byte boundary on, so that lines are written whole, and the values before it one by
// one: the gradient of 2,000 rows of 50,001 f32 values by stores past the caches 157 us, without
// it 175.  A distillation step, which waits for its sums between the passes, loses by the extra
// step: 1,023 rows of 32,001 f32 values 77 us and 73, 4,096 x 131,072 bf16 548 and 503.
template <typename T, int N, int U, int W, bool STREAM, bool LINES, typename F>
__device__ __forceinline__ void map_row(const T* z, T* d, int lo, int hi, int w, int lane, F f) {
  if constexpr (N > 1 && LINES) {
    int head = static_cast<int>(-reinterpret_cast<uintptr_t>(d + lo) % 64 / sizeof(T));
    if (head > hi - lo) head = hi - lo;
    if (w * 64 + lane < head) from_f(d[lo + w * 64 + lane], f(to_f(z[lo + w * 64 + lane])));
    lo += head;
  }
  const int nv = (hi - lo) / N;
  constexpr int STEP = W * 64 * U;
  for (int v0 = w * 64 + lane; v0 < nv; v0 += STEP) {
    float x[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v0 + u * W * 64 < nv) load_vec<N>(z + lo + (v0 + u * W * 64) * N, x[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v0 + u * W * 64 >= nv) break;
#pragma unroll
      for (int i = 0; i < N; ++i) x[u][i] = f(x[u][i]);
      store_vec<N, STREAM>(d + lo + (v0 + u * W * 64) * N, x[u]);
    }
  }
  if constexpr (N > 1) {
    const int v = lo + nv * N + w * 64 + lane;
    if (v < hi) from_f(d[v], f(to_f(z[v])));
  }
}
template <typename T, int N, int W>
__device__ __forceinline__ void zero_row(T* d, int lo, int hi, int w, int lane) {
  const int nv = (hi - lo) / N;
  float x[N] = {};
  for (int v = w * 64 + lane; v < nv; v += W * 64) store_vec<N>(d + lo + v * N, x);
  if constexpr (N > 1) {
    const int v = lo + nv * N + w * 64 + lane;
    if (v < hi) from_f(d[v], 0.f);
  }
}

// How the elementwise passes split rows over groups of 4 waves: at least 2048 groups
// where the rows are long enough, of at least 4096 values each.
inline Split map_split(int64_t rows, int64_t V) {
  int64_t p = rows > 0 && rows < 2048 ? (2048 + rows - 1) / rows : 1;
  if (p > V / 4096) p = V / 4096;
  if (p < 2) return {1, static_cast<int>(V)};
  int64_t len = (V + p - 1) / p;
  len = (len + 511) / 512 * 512;
  return {static_cast<int>((V + len - 1) / len), static_cast<int>(len)};
}

// HIP takes fewer than 2^32 threads along a grid's x: blocks beyond that go over its y, and the last
// of them may be past the end.
inline dim3 grid_of(int64_t blocks, int threads) {
  const int64_t most = ((int64_t(1) << 32) - 1) / threads, y = (blocks + most - 1) / most;
  return dim3(static_cast<unsigned>((blocks + y - 1) / y), static_cast<unsigned>(y));
}

inline bool ids_ok(int bits) { return bits == 8 || bits == 32 || bits == 64; }
inline bool dtype_ok(int d) { return d >= 0 && d <= 2; }

}  // namespace

#define TOK_DISPATCH(dtype, CALL)                 \
  do {                                            \
    if ((dtype) == 0) { using T = float; CALL; }  \
    else if ((dtype) == 1) { using T = bf16_t; CALL; } \
    else { using T = f16_t; CALL; }               \
  } while (0)

#define TOK_CHECK_ROWS()                                                                                       \
  GHM_CHECK(dtype_ok(dtype), "dtype (0 f32, 1 bf16, 2 f16)");                                                  \
  GHM_CHECK(rows >= 0 && rows < (int64_t(1) << 31) && V >= 1 && V <= (int64_t(1) << 30), "shape (rows < 2^31, V <= 2^30)"); \
  GHM_CHECK(n_inner >= 1 && s_outer >= 0 && s_inner >= 0, "row strides")
