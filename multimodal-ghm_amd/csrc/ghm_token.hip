// Token operators over a vocabulary of any size: log probabilities of given
// tokens with entropy and top alternatives, distillation from a teacher's top
// logits, and the scaled embedding lookup with its gradient.
//
// Logits rows are addressed as base + (r / n_inner) * s_outer + (r % n_inner) * s_inner
// elements, so a view past leading positions ([N][T][V] from position P on) is read
// in place.  Values are f32, bf16 or f16; every sum, maximum and statistic is f32.
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
// -inf; a difference is cut at -1e4 where it is a factor (e^-1e4 = 0).  NaN and +inf
// make s NaN.  c1, c2 carry log2 e.
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
  const float dm = fmaxf(a.m - m, -1e4f), f = __builtin_amdgcn_exp2f(dm * c1);
  const float n = dm == 0.f ? 0.f : a.n;  // what was at the old maximum joins the sums
  if constexpr (SECOND == SECOND_ENT) a.t = f * (a.t + dm * (a.s + n));
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

// emit(rank, key) for the k largest values of the group's range (key 0 past the last one
// if it holds fewer): the noted vectors at or above the last bound are ranked, then the
// values of the k best that reach the k-th vector's maximum.
template <typename T, int N, int W, typename F>
__device__ __forceinline__ void top_finish(const T* z, int lo, int hi, TopLds<N, W>* lds, TopState top, int k, int w,
                                           int lane, F emit) {
  uint64_t* cand = lds->cand + w * TOP_CAP;
  if (top.cnt > 64) {
    top_prune(cand, lds->merged + w * 64, top.cnt, k, lane);
    top.cnt = k;
  }
  group_sync<W>();  // every wave's last bound is there
  uint32_t bound = top.bound;
  if constexpr (W > 1) {
#pragma unroll
    for (int i = 0; i < W; ++i) bound = lds->bound[i] < bound ? lds->bound[i] : bound;
  }
  if (bound <= 0x00800000u) bound = 0;
  const uint64_t mine = lane < top.cnt ? cand[lane] : 0;
  const bool in = lane < top.cnt && static_cast<uint32_t>(mine >> 32) >= bound;
  const uint64_t mask = __ballot(in);
  int base = 0, all = __popcll(mask);
  if constexpr (W > 1) {
    if (lane == 0) lds->count[w] = all;
    if (w == 0 && lane == 0) lds->n_vals = 0;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      base += i < w ? lds->count[i] : 0;
      all += lds->count[i];
    }
  } else if (lane == 0) {
    lds->n_vals = 0;
  }
  if (in) lds->merged[base + __popcll(mask & ((uint64_t(1) << lane) - 1))] = mine;
  group_sync<W>();
  const int at = w * 64 + lane;
  if (at < all) {
    const uint64_t key = lds->merged[at];
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < all; ++i) rank += lds->merged[i] > key;
    if constexpr (N == 1) {
      if (rank < k) emit(rank, (key & 0xffffffff00000000ull) | (static_cast<uint32_t>(key) - lo));
    } else {
      if (rank < k) lds->best[rank] = key;
    }
  }
  if constexpr (N == 1) {
    for (int j = all + at; j < k; j += W * 64) emit(j, uint64_t(0));
  } else {
    group_sync<W>();
    const int nb = all < k ? all : k;
    const uint32_t least = all < k ? 0 : static_cast<uint32_t>(lds->best[k - 1] >> 32);
    for (int i = at; i < nb * N; i += W * 64) {
      const int id = lo + static_cast<int>(0xffffffffu - static_cast<uint32_t>(lds->best[i / N])) * N + i % N;
      if (id < hi) {
        const uint64_t key = top_key(to_f(z[id]), id);
        if (static_cast<uint32_t>(key >> 32) >= least) lds->vals[atomicAdd(&lds->n_vals, 1)] = key;
      }
    }
    group_sync<W>();
    const int n = lds->n_vals;
    for (int i = at; i < n; i += W * 64) {
      const uint64_t key = lds->vals[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank += lds->vals[j] > key;
      if (rank < k) emit(rank, key);
    }
    for (int j = n + at; j < k; j += W * 64) emit(j, uint64_t(0));
  }
}

// The same by k searches of the whole range, for one that holds NaN or +inf.
template <typename T, int N, int W, typename F>
__device__ __forceinline__ void top_search(const T* z, int lo, int hi, TopLds<N, W>* lds, int k, int w, int lane,
                                           F emit) {
  uint64_t last = ~uint64_t(0);
  for (int j = 0; j < k; ++j) {
    uint64_t best = 0;
    for (int v = lo + w * 64 + lane; v < hi; v += W * 64) {
      const uint64_t key = top_key(to_f(z[v]), v);
      best = key < last && key > best ? key : best;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      const uint64_t other = __shfl_xor(best, o, 64);
      best = other > best ? other : best;
    }
    if constexpr (W > 1) {
      if (lane == 0) lds->merged[w] = best;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < W; ++i) best = lds->merged[i] > best ? lds->merged[i] : best;
      __syncthreads();
    }
    if (w == 0 && lane == 0) emit(j, best);
    last = best;
  }
}

// ---------------------------------------------------------------------------
// Scores: m = max z, s = sum e^(z - m), log p_v = (z_v - m) - log s,
// H = log s - sum e^(z - m) (z - m) / s.  A value of -inf has probability 0 and
// adds nothing; a row without a finite maximum has no distribution (NaN).
// ---------------------------------------------------------------------------
struct ScoreOut {
  float *logprob, *entropy;
  float2* stats;
  float* top_lp;
  int64_t* top_id;
  int top_k;
};
__device__ __forceinline__ void score_padding(const ScoreOut& o, int64_t r, int at, int step) {
  if (at == 0) {
    o.logprob[r] = 0.f;
    if (o.entropy) o.entropy[r] = 0.f;
    if (o.stats) o.stats[r] = make_float2(0.f, 0.f);
  }
  for (int j = at; j < o.top_k; j += step) {
    o.top_lp[r * o.top_k + j] = 0.f;
    o.top_id[r * o.top_k + j] = -1;
  }
}
// zy: the target's logit, NaN for a target outside the vocabulary
__device__ __forceinline__ void score_write(const ScoreOut& o, int64_t r, const Sums& a, float ls, float zy) {
  if (o.logprob) o.logprob[r] = (zy - a.m) - ls;
  if (o.entropy) o.entropy[r] = ls - a.t / a.total();
  if (o.stats) o.stats[r] = make_float2(a.m, ls);
}
__device__ __forceinline__ void score_top(const ScoreOut& o, int64_t r, int j, uint64_t key, float m, float ls) {
  o.top_id[r * o.top_k + j] = 0xffffffffu - static_cast<uint32_t>(key);
  o.top_lp[r * o.top_k + j] = (key_value(key) - m) - ls;
}

// Groups of W waves take a row, or one of `parts` ranges of `part_len` values of it
// (part_sums != NULL: what they found goes there for k_score_join).
template <typename T, int N, int U, int W, bool TOP>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W, 4) void k_score(Rows rows, int64_t n_rows, int V, Ids targets,
                                                                 int64_t ignore, ScoreOut out, int parts, int part_len,
                                                                 float4* __restrict__ part_sums,
                                                                 uint64_t* __restrict__ part_keys) {
  constexpr int G = W == 1 ? 4 : 1;
  __shared__ float slots[W == 1 ? 1 : 3 * W];
  __shared__ TopLds<N, TOP ? W : 1> top_lds[TOP ? G : 1];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, w = wave % W;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * G + wave / W;
  const int64_t r = part_sums ? item / parts : item;
  if (r >= n_rows) return;
  const int64_t y = targets.p ? ld_id(targets, r) : 0;
  if (targets.p && y == ignore) {  // padding: nothing of the row is read
    if (!part_sums) score_padding(out, r, w * 64 + lane, W * 64);
    return;
  }
  const T* z = row_ptr<T>(rows, r);
  int lo = 0, hi = V;
  if (part_sums) {
    lo = static_cast<int>(item % parts) * part_len;
    hi = lo + part_len < V ? lo + part_len : V;
  }
  float zy = __builtin_nanf("");
  if (!part_sums && y >= 0 && y < V) zy = to_f(z[y]);
  TopLds<N, W>* lds = nullptr;
  if constexpr (TOP) lds = top_lds + wave / W;
  TopState top;
  Sums a = scan_row<T, N, U, W, SECOND_ENT, TOP>(z, lo, hi, LOG2E, LOG2E, w, lane, out.top_k, lds, top);
  a = group_join<SECOND_ENT, W>(a, slots, w, LOG2E, LOG2E);
  const float ls = a.log_s();
  if (part_sums) {
    if (w == 0 && lane == 0) part_sums[item] = make_float4(a.m, a.s, a.t, 0.f);
  } else if (w == 0 && lane == 0) {
    score_write(out, r, a, ls, zy);
  }
  if constexpr (TOP) {
    const auto emit = [&](int j, uint64_t key) {
      if (part_sums) part_keys[item * out.top_k + j] = key;
      else score_top(out, r, j, key, a.m, ls);
    };
    if (a.s == a.s) top_finish<T>(z, lo, hi, lds, top, out.top_k, w, lane, emit);
    else top_search<T>(z, lo, hi, lds, out.top_k, w, lane, emit);
  }
}

// One block per row joins at most 64 parts: lane p of every wave holds part p's sums; an
// alternative is at or above K, the ceil(k / q)-th largest of the parts' q-th entries,
// q = ceil(k / parts).
constexpr int MAX_PARTS = 64;
template <typename T>
__global__ __launch_bounds__(256) void k_score_join(Rows rows, int V, Ids targets, int64_t ignore, ScoreOut out,
                                                    int parts, const float4* __restrict__ part_sums,
                                                    const uint64_t* __restrict__ part_keys) {
  __shared__ uint64_t list[MAX_PARTS * GHM_TOP_MAX];
  __shared__ int n_list;
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int64_t y = targets.p ? ld_id(targets, r) : 0;
  if (targets.p && y == ignore) {
    score_padding(out, r, threadIdx.x, 256);
    return;
  }
  if (threadIdx.x == 0) n_list = 0;
  Sums a;
  if (lane < parts) {
    const float4 v = part_sums[r * parts + lane];
    a.m = v.x, a.s = v.y, a.t = v.z;
  }
  rebase<SECOND_ENT>(a, wave_max(a.m), LOG2E, LOG2E);
  a.s = wave_sum(a.s);
  a.t = wave_sum(a.t);
  const float ls = a.log_s();
  if (threadIdx.x == 0)
    score_write(out, r, a, ls, y >= 0 && y < V ? to_f(row_ptr<T>(rows, r)[y]) : __builtin_nanf(""));
  const int k = out.top_k;
  if (k == 0) return;
  const uint64_t* keys = part_keys + r * parts * k;
  const int q = (k + parts - 1) / parts;
  const uint32_t K = kth_bits(lane < parts ? static_cast<uint32_t>(keys[lane * k + q - 1] >> 32) : 0, (k + q - 1) / q);
  __syncthreads();
  for (int i = threadIdx.x; i < parts * k; i += 256) {
    const uint64_t key = keys[i];
    if (key != 0 && static_cast<uint32_t>(key >> 32) >= K) list[atomicAdd(&n_list, 1)] = key;
  }
  __syncthreads();
  const int n = n_list;
  for (int i = threadIdx.x; i < n; i += 256) {
    const uint64_t key = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list[j] > key;
    if (rank < k) score_top(out, r, rank, key, a.m, ls);
  }
}

// Rows of at most SHORT_V values: one lane per row, the row in registers, the
// alternatives by k searches.
constexpr int SHORT_V = 32;
template <typename T, int M>
__global__ __launch_bounds__(256) void k_score_short(Rows rows, int64_t n_rows, int V, Ids targets, int64_t ignore,
                                                     ScoreOut out) {
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (r >= n_rows) return;
  const int64_t y = targets.p ? ld_id(targets, r) : 0;
  if (targets.p && y == ignore) {
    score_padding(out, r, 0, 1);
    return;
  }
  const T* z = row_ptr<T>(rows, r);
  float x[M];
  Sums a;
#pragma unroll
  for (int v = 0; v < M; ++v) {
    x[v] = v < V ? to_f(z[v]) : NEG_INF;
    a.m = fmaxf(a.m, x[v]);
  }
  fold<SECOND_ENT, true>(a, x, LOG2E, LOG2E);
  float zy = __builtin_nanf("");
#pragma unroll
  for (int v = 0; v < M; ++v)
    if (v == y && v < V) zy = x[v];
  const float ls = a.log_s();
  score_write(out, r, a, ls, zy);
  uint32_t left = V < 32 ? (1u << V) - 1 : 0xffffffffu;
  for (int j = 0; j < out.top_k; ++j) {
    uint64_t best = 0;
#pragma unroll
    for (int v = 0; v < M; ++v) {
      const uint64_t key = top_key(x[v], v);
      if (((left >> v) & 1) && key > best) best = key;
    }
    left &= ~(1u << (0xffffffffu - static_cast<uint32_t>(best)));
    score_top(out, r, j, best, a.m, ls);
  }
}

// How a row is split (both kinds of logits operator): rows few and long go in parts so
// that about 512 groups are at work, each with at least one vector per lane of 8 waves.
struct Split {
  int parts, len;
};
inline bool one_wave(int64_t rows, int64_t V, int N) {
  return V <= 256 * N || (V <= 1536 * N && rows >= 1024);
}
inline Split row_split(int64_t rows, int64_t V) {
  const int64_t most = V / 4096;
  int64_t p = rows > 0 && rows < 512 ? (512 + rows - 1) / rows : 1;
  if (p > most) p = most;
  if (p > MAX_PARTS) p = MAX_PARTS;
  if (p < 2) return {1, static_cast<int>(V)};
  int64_t len = (V + p - 1) / p;
  len = (len + 511) / 512 * 512;
  return {static_cast<int>((V + len - 1) / len), static_cast<int>(len)};
}

// f(value, index) over a row's values lo .. hi - 1, written to d: batches of U vectors
template <typename T, int N, int U, int W, bool STREAM, typename F>
__device__ __forceinline__ void map_row(const T* z, T* d, int lo, int hi, int w, int lane, F f) {
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

// dz_v = -p_v [g_lp + sum_j g_top_j + g_H (log p_v + H)] + g_lp [v = y] + sum_j g_top_j [v = id_j]
struct ScoreGrad {
  const int64_t* top_id;
  const float2* stats;
  const float *entropy, *g_lp, *g_ent, *g_top;
  int top_k;
};
struct ScoreRow {  // the gradient at a value z other than the target and the alternatives
  float m, c, gs, g2, gh;
  __device__ __forceinline__ float operator()(float z) const {
    const float d = z - m;
    return -__builtin_amdgcn_exp2f(__builtin_fmaf(d, LOG2E, c)) * __builtin_fmaf(g2, fmaxf(d, -1e4f), gh);
  }
};
__device__ __forceinline__ ScoreRow score_row(const ScoreGrad& g, int64_t r, float g1, float top_sum) {
  ScoreRow o;
  const float2 st = g.stats[r];
  o.m = st.x;
  o.c = -st.y * LOG2E;
  o.gs = g1 + top_sum;
  o.g2 = g.g_ent ? g.g_ent[r] : 0.f;
  o.gh = g.g_ent ? __builtin_fmaf(o.g2, g.entropy[r] - st.y, o.gs) : o.gs;
  return o;
}

// the whole row part is written first, then the target's and the alternatives' entries again
template <typename T, int N, int U, int W>
__global__ __launch_bounds__(256) void k_score_bwd(Rows rows, int64_t n_rows, int V, Ids targets, int64_t ignore,
                                                   ScoreGrad g, int parts, int part_len, T* __restrict__ dz) {
  constexpr int G = 4 / W;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, w = wave % W;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * G + wave / W, r = item / parts;
  if (r >= n_rows) return;
  const int lo = static_cast<int>(item % parts) * part_len, hi = lo + part_len < V ? lo + part_len : V;
  T* d = dz + r * V;
  const int64_t y = targets.p ? ld_id(targets, r) : -1;
  if (targets.p && y == ignore) {
    zero_row<T, N, W>(d, lo, hi, w, lane);
    return;
  }
  const T* z = row_ptr<T>(rows, r);
  float g1 = g.g_lp ? g.g_lp[r] : 0.f;
  if (g.g_lp && (y < 0 || y >= V)) g1 = __builtin_nanf("");
  float top = 0.f;
  if (g.g_top) top = wave_sum(lane < g.top_k ? g.g_top[r * g.top_k + lane] : 0.f);
  const ScoreRow f = score_row(g, r, g1, top);
  map_row<T, N, U, W, false>(z, d, lo, hi, w, lane, f);
  group_sync<W>();
  if (w != 0) return;
  const int64_t id = g.g_top && lane < g.top_k ? g.top_id[r * g.top_k + lane] : -1;
  if (id >= lo && id < hi)
    from_f(d[id], f(to_f(z[id])) + g.g_top[r * g.top_k + lane] + (g.g_lp && id == y ? g1 : 0.f));
  if (g.g_lp && y >= lo && y < hi && __ballot(id == y) == 0 && lane == 0) from_f(d[y], f(to_f(z[y])) + g1);
}

template <typename T, int M>
__global__ __launch_bounds__(256) void k_score_bwd_short(Rows rows, int64_t n_rows, int V, Ids targets, int64_t ignore,
                                                         ScoreGrad g, T* __restrict__ dz) {
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (r >= n_rows) return;
  T* d = dz + r * V;
  const int64_t y = targets.p ? ld_id(targets, r) : -1;
  if (targets.p && y == ignore) {
    for (int v = 0; v < V; ++v) from_f(d[v], 0.f);
    return;
  }
  const T* z = row_ptr<T>(rows, r);
  float x[M], own[M];
#pragma unroll
  for (int v = 0; v < M; ++v) {
    x[v] = v < V ? to_f(z[v]) : 0.f;
    own[v] = 0.f;
  }
  float g1 = g.g_lp ? g.g_lp[r] : 0.f, top = 0.f;
  if (g.g_lp && (y < 0 || y >= V)) g1 = __builtin_nanf("");
  if (g.g_top)
    for (int j = 0; j < g.top_k; ++j) {
      const float t = g.g_top[r * g.top_k + j];
      const int64_t id = g.top_id[r * g.top_k + j];
      top += t;
#pragma unroll
      for (int v = 0; v < M; ++v) own[v] += v == id ? t : 0.f;
    }
  const ScoreRow f = score_row(g, r, g1, top);
#pragma unroll
  for (int v = 0; v < M; ++v)
    if (v < V) from_f(d[v], f(x[v]) + own[v] + (g.g_lp && v == y ? g1 : 0.f));
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

// ---------------------------------------------------------------------------
// Distillation: q = softmax(t / tau) over a row's present alternatives (id >= 0,
// logit above -inf), p = softmax(z / tau):
//   loss_r = (1 - a) (log s_1 - (z_y - m)) + a tau^2 sum_j q_j (log q_j - log p_{id_j})
//   dz_v = scale [(1 - a) (softmax(z)_v - [v = y]) + a tau (p_v - sum_{j: id_j = v} q_j)]
// ---------------------------------------------------------------------------
struct Teacher {
  Ids ids;
  const void* logits;
  int dtype, k;
};
__device__ __forceinline__ float ld_teacher(const Teacher& t, int64_t i) {
  if (t.dtype == 0) return static_cast<const float*>(t.logits)[i];
  if (t.dtype == 1) return to_f(static_cast<const bf16_t*>(t.logits)[i]);
  return to_f(static_cast<const f16_t*>(t.logits)[i]);
}
__device__ __forceinline__ bool teacher_has(const Teacher& t, int64_t i) {
  return ld_id(t.ids, i) >= 0 && !(ld_teacher(t, i) == NEG_INF);
}
// rows that count: the target is not the ignored one; without targets, an alternative is
// present.  Asked by the whole group, answered alike in every lane.
__device__ __forceinline__ bool row_counts(const Teacher& t, const Ids& targets, int64_t ignore, int64_t r, int lane) {
  if (targets.p) return ld_id(targets, r) != ignore;
  for (int j = lane; j - lane < t.k; j += 64)
    if (__ballot(j < t.k && teacher_has(t, r * t.k + j))) return true;
  return false;
}

struct Mix {  // c1: exponent factor of the row's first sum (log2 e, or log2 e / tau); c2 of the second
  float tau, it, alpha, c1, c2;
  bool hard, two;  // two: the hard labels' softmax and the teacher's are different ones
};
// what scales the gradient: grad_scale * upstream / counted rows
struct Upstream {
  const int* counts;  // counted rows per block of k_distill_count
  int n_counts;
  const float* norm;
  const float* up;
  int up_rows;
  float scale;
};
__device__ __forceinline__ float upstream(const Upstream& u, int64_t r, int lane) {
  float s = u.scale;
  if (u.counts) {
    int c = lane < u.n_counts ? u.counts[lane] : 0;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) c += __shfl_xor(c, o, 64);
    s *= 1.f / static_cast<float>(c > 1 ? c : 1);
  }
  if (u.norm) s *= u.norm[0];
  if (u.up) s *= u.up[u.up_rows ? r : 0];
  return s;
}

constexpr int MAX_COUNTS = 64;
__global__ __launch_bounds__(256) void k_distill_count(Teacher t, Ids targets, int64_t ignore, int64_t n, int64_t per,
                                                       int* __restrict__ counts) {
  __shared__ int red[4];
  const int64_t lo = blockIdx.x * per, hi = lo + per < n ? lo + per : n;
  int c = 0;
  for (int64_t r = lo + threadIdx.x; r < hi; r += 256) {
    bool in = false;
    if (targets.p) {
      in = ld_id(targets, r) != ignore;
    } else {
      for (int j = 0; j < t.k && !in; ++j) in = teacher_has(t, r * t.k + j);
    }
    c += in;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) c += __shfl_xor(c, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) counts[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// the sum of row losses and the number of counted rows of one range of rows, in a fixed
// order; a single block (or the second stage, over the ranges' results) writes the loss
__device__ __forceinline__ void distill_result(float s, int c, int mean, float* loss, float* norm) {
  const float inv = 1.f / static_cast<float>(c > 1 ? c : 1);
  if (mean) norm[0] = inv;
  loss[0] = mean ? s * inv : s;
}
__global__ __launch_bounds__(1024) void k_distill_total(const float* __restrict__ row_loss,
                                                        const float4* __restrict__ row_stats, int64_t n, int64_t per,
                                                        float2* __restrict__ parts, int mean,
                                                        float* __restrict__ loss, float* __restrict__ norm) {
  __shared__ float rs[16];
  __shared__ int rc[16];
  const int64_t lo = blockIdx.x * per, hi = lo + per < n ? lo + per : n;
  float s = 0.f;
  int c = 0;
#pragma unroll 8
  for (int64_t r = lo + threadIdx.x; r < hi; r += 1024) {
    s += row_loss[r];
    c += row_stats[r].w != 0.f;
  }
  s = wave_sum(s);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) c += __shfl_xor(c, o, 64);
  if ((threadIdx.x & 63) == 0) {
    rs[threadIdx.x >> 6] = s;
    rc[threadIdx.x >> 6] = c;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  s = 0.f, c = 0;
  for (int i = 0; i < 16; ++i) {
    s += rs[i];
    c += rc[i];
  }
  if (gridDim.x == 1) distill_result(s, c, mean, loss, norm);
  else parts[blockIdx.x] = make_float2(s, __int_as_float(c));
}
__global__ __launch_bounds__(64) void k_distill_total2(const float2* __restrict__ parts, int n, int mean,
                                                       float* __restrict__ loss, float* __restrict__ norm) {
  const float2 v = static_cast<int>(threadIdx.x) < n ? parts[threadIdx.x] : make_float2(0.f, 0.f);
  const float s = wave_sum(v.x);
  int c = __float_as_int(v.y);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) c += __shfl_xor(c, o, 64);
  if (threadIdx.x == 0) distill_result(s, c, mean, loss, norm);
}

// A row's teacher in LDS: ids (-1 absent) and q; log q = (t - mt) it - lt.  The entries take
// 8 k bytes per group of the launch's dynamic LDS (room for 1,024 of them in every block
// halved the waves per CU of short rows), group g's after those of the groups before.
template <int W>
struct TeacherLds {
  int* id;
  float *q, *slots;
};
extern __shared__ float teacher_lds[];
template <int W>
__device__ __forceinline__ TeacherLds<W> teacher_at(int group, int k, float* slots) {
  float* at = teacher_lds + 2 * k * group;
  return {reinterpret_cast<int*>(at), at + k, slots};
}
struct TeacherRow {
  float mt, lt;
  bool some, bad;  // an entry is present; one lies outside the vocabulary
};
template <int W>
__device__ __forceinline__ TeacherRow teacher_row(const Teacher& t, int64_t r, int V, float it, const TeacherLds<W>& lds,
                                                  int w, int lane) {
  TeacherRow o;
  float mt = -FLT_MAX, bad = 0.f;
  for (int j = w * 64 + lane; j < t.k; j += W * 64) {
    const int64_t id = ld_id(t.ids, r * t.k + j);
    const float x = ld_teacher(t, r * t.k + j);
    const bool has = id >= 0 && !(x == NEG_INF);
    if (has && id >= V) bad = 1.f;
    lds.id[j] = has && id < V ? static_cast<int>(id) : -1;
    lds.q[j] = has ? x : NEG_INF;
    if (has) mt = fmaxf(mt, x);
  }
  o.mt = group_max<W>(mt, lds.slots, w);
  float s = 0.f;
  for (int j = w * 64 + lane; j < t.k; j += W * 64) s += __builtin_amdgcn_exp2f((lds.q[j] - o.mt) * it * LOG2E);
  s = group_sum<W>(s, lds.slots + W, w);
  o.bad = group_max<W>(bad, lds.slots + 2 * W, w) != 0.f;
  o.some = s != 0.f;
  o.lt = logf(s);
  for (int j = w * 64 + lane; j < t.k; j += W * 64)
    lds.q[j] = o.some ? __builtin_amdgcn_exp2f(((lds.q[j] - o.mt) * it - o.lt) * LOG2E) : 0.f;
  group_sync<W>();
  return o;
}

// the loss of a row from its sums and its teacher; y checked by the caller's group
template <typename T, int W>
__device__ __forceinline__ float distill_row_loss(const T* z, int V, const Teacher& tc, int64_t r, const Mix& mix,
                                                  const TeacherRow& tr, const TeacherLds<W>& lds, float m, float l1, float l2,
                                                  int64_t y, int w, int lane) {
  float kl = 0.f;
  for (int j = w * 64 + lane; j < tc.k; j += W * 64) {
    const int id = lds.id[j];
    const float q = lds.q[j];
    if (id >= 0 && !(q == 0.f))
      kl += q * (((ld_teacher(tc, r * tc.k + j) - tr.mt) * mix.it - tr.lt) - ((to_f(z[id]) - m) * mix.it - l2));
  }
  kl = group_sum<W>(kl, lds.slots + 3 * W, w);
  float loss = mix.alpha == 0.f ? 0.f : mix.alpha * mix.tau * mix.tau * kl;
  if (mix.hard) loss += (1.f - mix.alpha) * (y >= 0 && y < V ? l1 - (to_f(z[y]) - m) : 0.f);
  return loss;
}

// The gradient of a row: the two softmaxes everywhere, then the teacher's and the target's
// entries again.
struct DistillGrad {
  float A, B, m, e, k, k1, AB;  // e, k: the teacher's exponent factor and offset, or the only one's
  bool two, none;
  __device__ __forceinline__ float one(float x) const { return AB * __builtin_amdgcn_exp2f(__builtin_fmaf(x - m, e, k)); }
  __device__ __forceinline__ float both(float x) const {
    const float d = x - m;
    return __builtin_fmaf(A, __builtin_amdgcn_exp2f(__builtin_fmaf(d, e, k)),
                          B * __builtin_amdgcn_exp2f(__builtin_fmaf(d, LOG2E, k1)));
  }
};
__device__ __forceinline__ DistillGrad distill_grad(const Mix& mix, bool some, float m, float l1, float l2, float scale) {
  DistillGrad g;
  g.A = some && mix.alpha != 0.f ? scale * mix.alpha * mix.tau : 0.f;
  g.B = mix.hard ? scale * (1.f - mix.alpha) : 0.f;
  g.AB = g.A + g.B;
  g.m = m;
  g.k1 = -l1 * LOG2E;
  // one exponential where the softmaxes are the same one, or only one of them counts
  const bool hard_only = !mix.two && g.A == 0.f && mix.hard;
  g.e = hard_only ? LOG2E : mix.c2;
  g.k = hard_only ? g.k1 : -l2 * LOG2E;
  g.two = mix.two;
  g.none = g.A == 0.f && g.B == 0.f && scale == scale;
  return g;
}
// the entries among values lo .. hi - 1, after the group's stores (a repeated id writes its
// sum each time)
template <typename T, int W>
__device__ __forceinline__ void distill_entries(const T* z, T* d, int lo, int hi, const Teacher& tc, const Mix& mix,
                                                const DistillGrad& g, const TeacherLds<W>& lds, int64_t y, int w,
                                                int lane) {
  const auto entry = [&](int id) {
    const float x = to_f(z[id]);
    float v = g.two ? g.both(x) : g.one(x), q = 0.f;
    for (int j = 0; j < tc.k; ++j) q += lds.id[j] == id ? lds.q[j] : 0.f;
    v -= g.A * q;
    if (id == y) v -= g.B;
    from_f(d[id], v);
  };
  for (int j = w * 64 + lane; j < tc.k; j += W * 64)
    if (lds.id[j] >= lo && lds.id[j] < hi) entry(lds.id[j]);
  if (mix.hard && y >= lo && y < hi && w == 0 && lane == 0) entry(static_cast<int>(y));
}
template <typename T, int N, int U, int W>
__device__ __forceinline__ void distill_row_grad(const T* z, T* d, int lo, int hi, const Teacher& tc, const Mix& mix,
                                                 const DistillGrad& g, const TeacherLds<W>& lds, int64_t y, int w,
                                                 int lane) {
  if (g.none) {
    zero_row<T, N, W>(d, lo, hi, w, lane);
    return;
  }
  if (g.two) map_row<T, N, U, W, true>(z, d, lo, hi, w, lane, [=](float x) { return g.both(x); });
  else map_row<T, N, U, W, true>(z, d, lo, hi, w, lane, [=](float x) { return g.one(x); });
  group_sync<W>();
  distill_entries<T, W>(z, d, lo, hi, tc, mix, g, lds, y, w, lane);
}

// Sums of a row, its loss, and its gradient if dz is there, by a group of W waves.
// row_stats: (m, log of the hard labels' sum, log of the teacher's, counted)
template <typename T, int N, int U, int W, bool TWO>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void k_distill(Rows rows, int64_t n_rows, int V, Teacher tc,
                                                                   Ids targets, int64_t ignore, Mix mix, Upstream up,
                                                                   float* __restrict__ row_loss,
                                                                   float4* __restrict__ row_stats,
                                                                   T* __restrict__ dz) {
  constexpr int G = W == 1 ? 4 : 1, SECOND = TWO ? SECOND_EXP : SECOND_NONE;
  __shared__ float slots[3 * W];
  __shared__ float teach_slots[G][4 * W];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, w = wave % W;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * G + wave / W;
  if (r >= n_rows) return;
  T* d = dz ? dz + r * V : nullptr;
  if (!row_counts(tc, targets, ignore, r, lane)) {
    if (w == 0 && lane == 0) {
      row_loss[r] = 0.f;
      row_stats[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (d) zero_row<T, N, W>(d, 0, V, w, lane);
    return;
  }
  const T* z = row_ptr<T>(rows, r);
  const int64_t y = targets.p ? ld_id(targets, r) : -1;
  TopState no;
  Sums a = scan_row<T, N, U, W, SECOND, false>(z, 0, V, mix.c1, mix.c2, w, lane, 0,
                                               static_cast<TopLds<N, W>*>(nullptr), no);
  const TeacherLds<W> lds = teacher_at<W>(wave / W, tc.k, teach_slots[wave / W]);
  const TeacherRow tr = teacher_row<W>(tc, r, V, mix.it, lds, w, lane);
  a = group_join<SECOND, W>(a, slots, w, mix.c1, mix.c2);
  const float l1 = a.log_s(), l2 = TWO ? a.log_t() : l1;
  float loss = distill_row_loss<T, W>(z, V, tc, r, mix, tr, lds, a.m, l1, l2, y, w, lane);
  const bool bad = tr.bad || (targets.p && (y < 0 || y >= V));
  if (w == 0 && lane == 0) {
    row_loss[r] = bad ? __builtin_nanf("") : loss;
    row_stats[r] = make_float4(a.m, l1, l2, 1.f);
  }
  if (d)
    distill_row_grad<T, N, U, W>(z, d, 0, V, tc, mix,
                                 distill_grad(mix, tr.some, a.m, l1, l2, bad ? __builtin_nanf("") : upstream(up, r, lane)),
                                 lds, y, w, lane);
}

// Packed values stay packed across this point: without it the compiler keeps the unpacked
// floats from one pass to the next, twice the registers of 16-bit values.
template <int R>
__device__ __forceinline__ void hold(u32x4 (&raw)[R]) {
#pragma unroll
  for (int u = 0; u < R; ++u) asm volatile("" : "+v"(raw[u]));
}

// The same with the row held in registers between the sums and the gradient (R vectors per
// lane, R * 64 * W * N values at most): the logits are read once.
template <typename T, int R, int W, bool TWO>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W, R == 16 ? 4 : 1) void k_distill_step(Rows rows, int64_t n_rows, int V, Teacher tc,
                                                                        Ids targets, int64_t ignore, Mix mix,
                                                                        Upstream up, float* __restrict__ row_loss,
                                                                        float4* __restrict__ row_stats,
                                                                        T* __restrict__ dz) {
  constexpr int G = W == 1 ? 4 : 1, N = Vec<T>::N, SECOND = TWO ? SECOND_EXP : SECOND_NONE;
  __shared__ float slots[3 * W];
  __shared__ float teach_slots[G][4 * W];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, w = wave % W;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * G + wave / W;
  if (r >= n_rows) return;
  T* d = dz + r * V;
  if (!row_counts(tc, targets, ignore, r, lane)) {
    if (w == 0 && lane == 0) {
      row_loss[r] = 0.f;
      row_stats[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    zero_row<T, N, W>(d, 0, V, w, lane);
    return;
  }
  const T* z = row_ptr<T>(rows, r);
  const int64_t y = targets.p ? ld_id(targets, r) : -1;
  // vectors as in scan_row: the last one of a row that does not divide is its last N values
  const int tail = V % N, nv = V / N + (tail ? 1 : 0), v0 = w * 64 + lane;
  u32x4 raw[R];
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int v = v0 + u * W * 64, at = v < nv ? v * N : V - N;
    raw[u] = *reinterpret_cast<const typename Vec<T>::raw*>(z + (at + N <= V ? at : V - N));
  }
  const TeacherLds<W> lds = teacher_at<W>(wave / W, tc.k, teach_slots[wave / W]);
  const TeacherRow tr = teacher_row<W>(tc, r, V, mix.it, lds, w, lane);
  Sums a;
#pragma unroll
  for (int u = 0; u < R; ++u) {  // values seen twice do not change a maximum
    float x[N];
    unpack<T>(raw[u], x);
#pragma unroll
    for (int i = 0; i < N; ++i) a.m = fmaxf(a.m, x[i]);
  }
  a.m = group_max<W>(a.m, slots, w);
  hold(raw);
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int v = v0 + u * W * 64;
    if (v - lane >= nv) break;
    float x[N];
    unpack<T>(raw[u], x);
    if (v - lane + 64 >= nv) {  // the wave's last vectors
      const int skip = v >= nv ? N : v == nv - 1 && tail ? N - tail : 0;
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = i < skip ? NEG_INF : x[i];
    }
    fold<SECOND, false>(a, x, mix.c1, mix.c2);
  }
  a.s = group_sum<W>(a.s, slots + W, w);
  if constexpr (TWO) a.t = group_sum<W>(a.t, slots + 2 * W, w);
  const float l1 = a.log_s(), l2 = TWO ? a.log_t() : l1;
  const float loss = distill_row_loss<T, W>(z, V, tc, r, mix, tr, lds, a.m, l1, l2, y, w, lane);
  const bool bad = tr.bad || (targets.p && (y < 0 || y >= V));
  if (w == 0 && lane == 0) {
    row_loss[r] = bad ? __builtin_nanf("") : loss;
    row_stats[r] = make_float4(a.m, l1, l2, 1.f);
  }
  const DistillGrad g = distill_grad(mix, tr.some, a.m, l1, l2, bad ? __builtin_nanf("") : upstream(up, r, lane));
  if (g.none) {
    zero_row<T, N, W>(d, 0, V, w, lane);
    return;
  }
  hold(raw);
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const int v = v0 + u * W * 64;
    if (v >= nv) break;
    float x[N];
    unpack<T>(raw[u], x);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = TWO ? g.both(x[i]) : g.one(x[i]);
    store_vec<N, true>(d + (v * N + N <= V ? v * N : V - N), x);
  }
  group_sync<W>();
  distill_entries<T, W>(z, d, 0, V, tc, mix, g, lds, y, w, lane);
}

// long rows, few of them: the sums of one part of a row ...
template <typename T, int N, int U, int W, bool TWO>
__global__ __launch_bounds__(64 * W) void k_distill_part(Rows rows, int V, Teacher tc, Ids targets, int64_t ignore,
                                                         Mix mix, int parts, int part_len,
                                                         float4* __restrict__ part_sums) {
  constexpr int SECOND = TWO ? SECOND_EXP : SECOND_NONE;
  __shared__ float slots[3 * W];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t r = blockIdx.x / parts;
  if (!row_counts(tc, targets, ignore, r, lane)) return;
  const int lo = static_cast<int>(blockIdx.x % parts) * part_len, hi = lo + part_len < V ? lo + part_len : V;
  TopState no;
  Sums a = scan_row<T, N, U, W, SECOND, false>(row_ptr<T>(rows, r), lo, hi, mix.c1, mix.c2, w, lane, 0,
                                               static_cast<TopLds<N, W>*>(nullptr), no);
  a = group_join<SECOND, W>(a, slots, w, mix.c1, mix.c2);
  if (threadIdx.x == 0) part_sums[blockIdx.x] = make_float4(a.m, a.s, a.t, 0.f);
}
// ... joined, with the loss ...
template <typename T, bool TWO>
__global__ __launch_bounds__(256) void k_distill_join(Rows rows, int V, Teacher tc, Ids targets, int64_t ignore,
                                                      Mix mix, int parts, const float4* __restrict__ part_sums,
                                                      float* __restrict__ row_loss, float4* __restrict__ row_stats) {
  constexpr int SECOND = TWO ? SECOND_EXP : SECOND_NONE;
  __shared__ float teach_slots[16];
  const TeacherLds<4> lds = teacher_at<4>(0, tc.k, teach_slots);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t r = blockIdx.x;
  if (!row_counts(tc, targets, ignore, r, lane)) {
    if (threadIdx.x == 0) {
      row_loss[r] = 0.f;
      row_stats[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    return;
  }
  const int64_t y = targets.p ? ld_id(targets, r) : -1;
  Sums a;
  if (lane < parts) {
    const float4 v = part_sums[r * parts + lane];
    a.m = v.x, a.s = v.y, a.t = v.z;
  }
  rebase<SECOND>(a, wave_max(a.m), mix.c1, mix.c2);
  a.s = wave_sum(a.s);
  if constexpr (TWO) a.t = wave_sum(a.t);
  const TeacherRow tr = teacher_row<4>(tc, r, V, mix.it, lds, w, lane);
  const float l1 = a.log_s(), l2 = TWO ? a.log_t() : l1;
  const float loss = distill_row_loss<T, 4>(row_ptr<T>(rows, r), V, tc, r, mix, tr, lds, a.m, l1, l2, y, w, lane);
  if (threadIdx.x == 0) {
    row_loss[r] = tr.bad || (targets.p && (y < 0 || y >= V)) ? __builtin_nanf("") : loss;
    row_stats[r] = make_float4(a.m, l1, l2, 1.f);
  }
}
// ... and the gradient from the row's statistics
template <typename T, int N, int U, int W>
__global__ __launch_bounds__(256) void k_distill_grad(Rows rows, int64_t n_rows, int V, Teacher tc, Ids targets,
                                                      int64_t ignore, Mix mix, Upstream up, int parts, int part_len,
                                                      const float4* __restrict__ row_stats, T* __restrict__ dz) {
  constexpr int G = 4 / W;
  __shared__ float teach_slots[G][4 * W];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, w = wave % W;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * G + wave / W, r = item / parts;
  if (r >= n_rows) return;
  const int lo = static_cast<int>(item % parts) * part_len, hi = lo + part_len < V ? lo + part_len : V;
  T* d = dz + r * V;
  const float4 st = row_stats[r];
  if (st.w == 0.f) {
    zero_row<T, N, W>(d, lo, hi, w, lane);
    return;
  }
  const int64_t y = targets.p ? ld_id(targets, r) : -1;
  const TeacherLds<W> lds = teacher_at<W>(wave / W, tc.k, teach_slots[wave / W]);
  const TeacherRow tr = teacher_row<W>(tc, r, V, mix.it, lds, w, lane);
  const bool bad = tr.bad || (targets.p && (y < 0 || y >= V));
  distill_row_grad<T, N, U, W>(
      row_ptr<T>(rows, r), d, lo, hi, tc, mix,
      distill_grad(mix, tr.some, st.x, st.y, st.z, bad ? __builtin_nanf("") : upstream(up, r, lane)), lds, y, w, lane);
}

// Rows of at most SHORT_V values, one lane per row: loss, statistics and gradient, each
// if asked for.
template <typename T, int M>
__global__ __launch_bounds__(256) void k_distill_short(Rows rows, int64_t n_rows, int V, Teacher tc, Ids targets,
                                                       int64_t ignore, Mix mix, Upstream up,
                                                       float* __restrict__ row_loss, float4* __restrict__ row_stats,
                                                       T* __restrict__ dz) {
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const bool live = r0 < n_rows;
  const int64_t r = live ? r0 : n_rows - 1;
  float scale = dz ? upstream(up, r, threadIdx.x & 63) : 0.f;  // by whole waves
  if (!live) return;
  const int64_t y = targets.p ? ld_id(targets, r) : -1;
  float mt = -FLT_MAX;
  bool some = false, bad = targets.p && (y < 0 || y >= V);
  for (int j = 0; j < tc.k; ++j) {
    if (!teacher_has(tc, r * tc.k + j)) continue;
    some = true;
    mt = fmaxf(mt, ld_teacher(tc, r * tc.k + j));
    if (ld_id(tc.ids, r * tc.k + j) >= V) bad = true;
  }
  if (targets.p ? y == ignore : !some) {
    if (row_loss) {
      row_loss[r] = 0.f;
      row_stats[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (dz)
      for (int v = 0; v < V; ++v) from_f(dz[r * V + v], 0.f);
    return;
  }
  const T* z = row_ptr<T>(rows, r);
  float x[M], q[M];
  Sums a;
#pragma unroll
  for (int v = 0; v < M; ++v) {
    x[v] = v < V ? to_f(z[v]) : NEG_INF;
    a.m = fmaxf(a.m, x[v]);
    q[v] = 0.f;
  }
  fold<SECOND_EXP, true>(a, x, LOG2E, mix.c2);
  const float l1 = a.log_s(), l2 = a.log_t();
  float st = 0.f, kl = 0.f;
  for (int j = 0; j < tc.k; ++j)
    if (teacher_has(tc, r * tc.k + j))
      st += __builtin_amdgcn_exp2f((ld_teacher(tc, r * tc.k + j) - mt) * mix.it * LOG2E);
  const float lt = logf(st);
  for (int j = 0; j < tc.k; ++j) {
    if (!teacher_has(tc, r * tc.k + j)) continue;
    const int64_t id = ld_id(tc.ids, r * tc.k + j);
    const float lq = (ld_teacher(tc, r * tc.k + j) - mt) * mix.it - lt, qj = __builtin_amdgcn_exp2f(lq * LOG2E);
    float zi = 0.f;
#pragma unroll
    for (int v = 0; v < M; ++v) {
      q[v] += v == id ? qj : 0.f;
      zi = v == id ? x[v] : zi;
    }
    if (!(qj == 0.f)) kl += qj * (lq - ((zi - a.m) * mix.it - l2));
  }
  if (row_loss) {
    float loss = mix.alpha == 0.f ? 0.f : mix.alpha * mix.tau * mix.tau * kl;
    float zy = 0.f;
#pragma unroll
    for (int v = 0; v < M; ++v) zy = v == y ? x[v] : zy;
    if (mix.hard) loss += (1.f - mix.alpha) * (l1 - (zy - a.m));
    row_loss[r] = bad ? __builtin_nanf("") : loss;
    row_stats[r] = make_float4(a.m, l1, l2, 1.f);
  }
  if (!dz) return;
  if (bad) scale = __builtin_nanf("");
  const float A = some && mix.alpha != 0.f ? scale * mix.alpha * mix.tau : bad ? scale : 0.f;
  const float B = mix.hard ? scale * (1.f - mix.alpha) : 0.f;
#pragma unroll
  for (int v = 0; v < M; ++v) {
    if (v >= V) break;
    const float d = x[v] - a.m;
    float g = A * (__builtin_amdgcn_exp2f(__builtin_fmaf(d, mix.it * LOG2E, -l2 * LOG2E)) - q[v]);
    if (mix.hard) g += B * (__builtin_amdgcn_exp2f(__builtin_fmaf(d, LOG2E, -l1 * LOG2E)) - (v == y ? 1.f : 0.f));
    from_f(dz[r * V + v], g);
  }
}

// ---------------------------------------------------------------------------
// Scaled embedding: out_i = scale W[tok_i].
// ---------------------------------------------------------------------------
// Rows of D values are taken in vectors of VE; the last one of a row that does not divide is
// its last VE values, shared with the vector before (both hold the same results).  Rows
// shorter than a vector go value by value.
template <int VE>
__device__ __forceinline__ int edge_col(int c, int D) {
  return c + VE <= D || D < VE ? c : D - VE;
}
template <typename T, int VE>
__device__ __forceinline__ void load_cols(const T* row, int c, int D, float (&x)[VE]) {
  if (D >= VE) {
    load_vec<VE>(row + c, x);
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) x[i] = c + i < D ? to_f(row[c + i]) : 0.f;
  }
}
template <typename T, int VE, bool STREAM = false>
__device__ __forceinline__ void store_cols(T* row, int c, int D, const float (&x)[VE]) {
  if (D >= VE) {
    store_vec<VE, STREAM>(row + c, x);
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (c + i < D) from_f(row[c + i], x[i]);
  }
}

// A block takes `per` rows of `vecs` vectors; lanes take vectors in turn.
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void k_embed_rows(Ids tok, const T* __restrict__ weight, int64_t w_stride,
                                                    float scale, T* __restrict__ out, int64_t N, int64_t V, int D,
                                                    int vecs, int per) {
  constexpr int VE = Vec<T>::N, U = 4;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * per;
  const int n = static_cast<int>(N - i0 < per ? N - i0 : per) * vecs;
  for (int t0 = threadIdx.x; t0 < n; t0 += 256 * U) {
    int64_t v[U];
    float x[U][VE];
    ld_ids<U>(tok, v, [&](int u) { return i0 + (t0 + 256 * u < n ? t0 + 256 * u : t0) / vecs; });
#pragma unroll
    for (int u = 0; u < U; ++u) {  // every load is issued before the first is waited for; a bad token reads row 0
      const int64_t row = v[u] >= 0 && v[u] < V ? v[u] : 0;
      load_cols<T, VE>(weight + row * w_stride, edge_col<VE>((t0 + 256 * u < n ? t0 + 256 * u : t0) % vecs * VE, D), D,
                       x[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + 256 * u;
      if (t >= n) break;
      const float f = v[u] >= 0 && v[u] < V ? scale : __builtin_nanf("");
#pragma unroll
      for (int i = 0; i < VE; ++i) x[u][i] *= f;
      store_cols<T, VE, STREAM>(out + (i0 + t / vecs) * D, edge_col<VE>(t % vecs * VE, D), D, x[u]);
    }
  }
}

// ---------------------------------------------------------------------------
// Its gradient dW_v = scale sum_{i: tok_i = v} dout_i.  The positions are sorted by token
// (stable radix sort, so a token's positions stay in order); chunks of the sorted list are
// summed in f32, a token that crosses chunks through partial rows joined in order; table
// rows without a token are written 0 beside it.  No atomics on values: a fixed order.
// ---------------------------------------------------------------------------
constexpr int SORT_BITS = 9, SORT_BINS = 1 << SORT_BITS, SORT_ROUNDS = 8;
constexpr int SORT_SELF_N = 16384;  // up to this many positions a block counts them all itself
constexpr int SORT_TILES = 128;     // up to this many tiles it sums their counts itself

__device__ __forceinline__ uint32_t digit(uint32_t key, int shift, int bits) { return (key >> shift) & ((1u << bits) - 1); }
// The sorted key of a position is its token, or `none` for a token that gets no gradient.
struct SortIn {  // the first pass reads tokens, later ones the previous pass's keys and positions
  Ids tok;
  const uint32_t *key, *pos;
  int64_t pad;
  uint32_t none;
};
// keys of positions i, i + step, ... (the last one's again past the end: no load waits for a branch)
template <int R>
__device__ __forceinline__ void sort_in(const SortIn& in, int64_t i, int64_t step, int64_t N, uint32_t (&key)[R]) {
  const auto at = [&](int q) { return i + q * step < N ? i + q * step : N - 1; };
  if (in.key) {
#pragma unroll
    for (int q = 0; q < R; ++q) key[q] = in.key[at(q)];
  } else {
    int64_t v[R];
    ld_ids<R>(in.tok, v, at);
#pragma unroll
    for (int q = 0; q < R; ++q) key[q] = v[q] >= 0 && v[q] < in.none && v[q] != in.pad ? static_cast<uint32_t>(v[q]) : in.none;
  }
}

// Table rows that have a token, one byte each: cleared by the first launch of a sort and set
// by a later one.
__device__ __forceinline__ void clear_used(uint32_t* used, int64_t words, int threads) {
  if (used)
    for (int64_t j = static_cast<int64_t>(blockIdx.x) * threads + threadIdx.x; j < words;
         j += static_cast<int64_t>(gridDim.x) * threads)
      used[j] = 0;
}

// counts[tile][digit]
template <int W>
__global__ __launch_bounds__(64 * W) void k_sort_count(SortIn in, int64_t N, int shift, int bits,
                                                       uint32_t* __restrict__ counts,
                                                       uint32_t* __restrict__ used, int64_t used_words) {
  __shared__ uint32_t bins[SORT_BINS];
  constexpr int TILE = 64 * W * SORT_ROUNDS;
  for (int d = threadIdx.x; d < SORT_BINS; d += 64 * W) bins[d] = 0;
  clear_used(used, used_words, 64 * W);
  __syncthreads();
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * TILE + threadIdx.x;
  uint32_t key[SORT_ROUNDS];
  sort_in<SORT_ROUNDS>(in, i0, 64 * W, N, key);
#pragma unroll
  for (int q = 0; q < SORT_ROUNDS; ++q)
    if (i0 + q * 64 * W < N) atomicAdd(&bins[digit(key[q], shift, bits)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < SORT_BINS; d += 64 * W) counts[static_cast<int64_t>(blockIdx.x) * SORT_BINS + d] = bins[d];
}
// many tiles: counts become, digit by digit, the sums over the tiles before; the totals follow
__global__ __launch_bounds__(64) void k_sort_scan(uint32_t* __restrict__ counts, int64_t tiles) {
  uint32_t* c = counts + blockIdx.x * 64 + threadIdx.x;
  uint32_t s = 0;
#pragma unroll 8
  for (int64_t t = 0; t < tiles; ++t) {
    const uint32_t v = c[t * SORT_BINS];
    c[t * SORT_BINS] = s;
    s += v;
  }
  c[tiles * SORT_BINS] = s;
}
// One pass: positions go to the start of their digit + the digit's count in earlier tiles +
// in earlier waves + in this wave's earlier rounds + among lower lanes.  A wave takes
// 64 * SORT_ROUNDS consecutive positions, so the sort is stable.  The counts per tile come
// from k_sort_count: summed here (SORT_SUM) or by k_sort_scan (SORT_SCANNED); for few
// positions each block counts all of them itself (SORT_SELF: one launch instead of two).
enum { SORT_SUM, SORT_SCANNED, SORT_SELF };
template <int W, int MODE>
__global__ __launch_bounds__(64 * W) void k_sort_scatter(SortIn in, int64_t N, int shift, int bits,
                                                         const uint32_t* __restrict__ counts, int tiles,
                                                         uint32_t* __restrict__ key_out, uint32_t* __restrict__ pos_out,
                                                         uint8_t* __restrict__ set_used, int one_pass,
                                                         uint32_t* __restrict__ clear, int64_t used_words) {
  // SORT_SUM: groups of 128 threads take 4 digits each of every GROUPS-th tile
  constexpr int GROUPS = MODE == SORT_SUM ? W / 2 : 1;
  __shared__ uint32_t tsum[2][GROUPS][MODE == SORT_SUM ? SORT_BINS : 1];
  // equal digits of a wave meet at one of SPREAD counters (64 lanes of 10 tokens at one each
  // took 14 us for 10,368 positions)
  constexpr int SPREAD = MODE == SORT_SELF ? 8 : 1;
  __shared__ uint32_t wbins[W][SORT_BINS], base[SORT_BINS], wsum[SORT_BINS / 64];
  __shared__ uint32_t self[2][MODE == SORT_SELF ? SORT_BINS * SPREAD : 1];
  constexpr int TILE = 64 * W * SORT_ROUNDS;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t i0 = (static_cast<int64_t>(blockIdx.x) * W + w) * 64 * SORT_ROUNDS + lane;
  uint32_t key[SORT_ROUNDS], at[SORT_ROUNDS], pos[SORT_ROUNDS];
  sort_in<SORT_ROUNDS>(in, i0, 64, N, key);
#pragma unroll
  for (int q = 0; q < SORT_ROUNDS; ++q) {
    const int64_t i = i0 + q * 64;
    pos[q] = in.pos ? in.pos[i < N ? i : N - 1] : static_cast<uint32_t>(i);
  }
  for (int d = lane; d < SORT_BINS; d += 64) wbins[w][d] = 0;
  clear_used(clear, used_words, 64 * W);
  if constexpr (MODE == SORT_SELF) {
    for (int d = threadIdx.x; d < SORT_BINS * SPREAD; d += 64 * W) self[0][d] = self[1][d] = 0;
    __syncthreads();
    for (int64_t t0 = 0; t0 < N; t0 += 2 * TILE) {
      uint32_t k[2 * SORT_ROUNDS];
      sort_in<2 * SORT_ROUNDS>(in, t0 + threadIdx.x, 64 * W, N, k);
#pragma unroll
      for (int q = 0; q < 2 * SORT_ROUNDS; ++q) {
        const int64_t i = t0 + threadIdx.x + q * 64 * W;
        const uint32_t d = digit(k[q], shift, bits) * SPREAD + lane % SPREAD;
        if (i < N) atomicAdd(&self[i < static_cast<int64_t>(blockIdx.x) * TILE ? 0 : 1][d], 1u);
      }
    }
  } else {
    wave_fence();
  }
  if constexpr (MODE == SORT_SUM) {
    u32x4 before = {}, all = {};
    const int d = (threadIdx.x & 127) * 4;
#pragma unroll 16
    for (int t = threadIdx.x >> 7; t < tiles; t += GROUPS) {
      const u32x4 c = *reinterpret_cast<const u32x4*>(counts + t * SORT_BINS + d);
      before += t < static_cast<int>(blockIdx.x) ? c : u32x4{};
      all += c;
    }
    *reinterpret_cast<u32x4*>(&tsum[0][threadIdx.x >> 7][d]) = before;
    *reinterpret_cast<u32x4*>(&tsum[1][threadIdx.x >> 7][d]) = all;
  }
#pragma unroll
  for (int q = 0; q < SORT_ROUNDS; ++q) {
    const bool live = i0 + q * 64 < N;
    const uint32_t d = digit(key[q], shift, bits);
    uint64_t same = __ballot(live);
    for (int bit = 0; bit < bits; ++bit) {
      const uint64_t m = __ballot((d >> bit) & 1);
      same &= (d >> bit) & 1 ? m : ~m;
    }
    const uint64_t lower = same & ((uint64_t(1) << lane) - 1);
    at[q] = wbins[w][d] + __popcll(lower);
    wave_fence();
    if (live && lower == 0) wbins[w][d] += __popcll(same);
    wave_fence();
  }
  __syncthreads();
  // counts become starts: over the waves, over earlier tiles, and by a scan over the digits
  for (int d = threadIdx.x; d < SORT_BINS; d += 64 * W) {
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const uint32_t c = wbins[j][d];
      wbins[j][d] = mine;
      mine += c;
    }
    uint32_t before = 0, all = 0;
    if constexpr (MODE == SORT_SELF) {
#pragma unroll
      for (int j = 0; j < SPREAD; ++j) {
        before += self[0][d * SPREAD + j];
        all += self[1][d * SPREAD + j];
      }
      all += before;
      if (one_pass && blockIdx.x == 0 && d < static_cast<int64_t>(in.none)) set_used[d] = all != 0;
    } else if constexpr (MODE == SORT_SCANNED) {
      before = counts[static_cast<int64_t>(blockIdx.x) * SORT_BINS + d];
      all = counts[static_cast<int64_t>(tiles) * SORT_BINS + d];
    } else {
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        before += tsum[0][j][d];
        all += tsum[1][j][d];
      }
    }
    uint32_t inc = all;  // 64 consecutive digits per wave
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t up = __shfl_up(inc, o, 64);
      inc += lane >= o ? up : 0;
    }
    if (lane == 63) wsum[d >> 6] = inc;
    base[d] = inc - all + before;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < SORT_BINS; d += 64 * W)
    for (int j = 0; j < d >> 6; ++j) base[d] += wsum[j];
  __syncthreads();
#pragma unroll
  for (int q = 0; q < SORT_ROUNDS; ++q) {
    if (i0 + q * 64 >= N) break;
    const uint32_t d = digit(key[q], shift, bits), to = base[d] + wbins[w][d] + at[q];
    key_out[to] = key[q];
    pos_out[to] = pos[q];
    if (set_used && !one_pass && key[q] != in.none) set_used[key[q]] = 1;
  }
}

// Up to SORT_ONE positions of a table of at most USED_ONE rows: all passes by one block,
// key and position in one word of LDS between them.
constexpr int ROUNDS = 4, POS_BITS = 12, SORT_ONE = 1 << POS_BITS, USED_ONE = (1 << (32 - POS_BITS)) - 1;
__global__ __launch_bounds__(1024) void k_sort_one(SortIn in, int N, int passes, int bits, uint32_t* __restrict__ key_out,
                                                   uint32_t* __restrict__ pos_out, uint32_t* __restrict__ used,
                                                   int used_words) {
  constexpr int W = 16;
  __shared__ uint32_t word[1024 * ROUNDS], wbins[W][SORT_BINS], base[SORT_BINS], wsum[SORT_BINS / 64];
  __shared__ uint16_t rank[1024 * ROUNDS];  // among the wave's equal digits
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, i0 = w * 64 * ROUNDS + lane;
  {
    uint32_t key[ROUNDS];
    sort_in<ROUNDS>(in, i0, 64, N, key);
    for (int j = threadIdx.x; j < used_words; j += 1024) used[j] = 0;
#pragma unroll
    for (int q = 0; q < ROUNDS; ++q) {
      const int i = i0 + q * 64;
      if (i < N) word[i] = key[q] << POS_BITS | i;
    }
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = POS_BITS + p * bits;
    for (int d = lane; d < SORT_BINS; d += 64) wbins[w][d] = 0;
    wave_fence();  // a wave ranks the words that it wrote, or that a barrier has passed
    for (int i = i0; i - lane < N && i < i0 + 64 * ROUNDS; i += 64) {
      const bool live = i < N;
      const uint32_t d = live ? digit(word[i], shift, bits) : 0;
      uint64_t same = __ballot(live);
      for (int bit = 0; bit < bits; ++bit) {
        const uint64_t m = __ballot((d >> bit) & 1);
        same &= (d >> bit) & 1 ? m : ~m;
      }
      const uint64_t lower = same & ((uint64_t(1) << lane) - 1);
      const uint32_t before = wbins[w][d];
      if (live) rank[i] = static_cast<uint16_t>(before + __popcll(lower));
      wave_fence();
      if (live && lower == 0) wbins[w][d] = before + __popcll(same);
      wave_fence();
    }
    __syncthreads();
    if (threadIdx.x < SORT_BINS) {  // counts become starts: over the waves, then over the digits
      const int d = threadIdx.x;
      uint32_t all = 0;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const uint32_t c = wbins[j][d];
        wbins[j][d] = all;
        all += c;
      }
      uint32_t inc = all;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = __shfl_up(inc, o, 64);
        inc += lane >= o ? up : 0;
      }
      if (lane == 63) wsum[d >> 6] = inc;
      base[d] = inc - all;
    }
    __syncthreads();
    if (threadIdx.x < SORT_BINS)
      for (int j = 0; j < static_cast<int>(threadIdx.x) >> 6; ++j) base[threadIdx.x] += wsum[j];
    __syncthreads();
    uint32_t x[ROUNDS], to[ROUNDS];
#pragma unroll
    for (int q = 0; q < ROUNDS; ++q) {
      const int i = i0 + q * 64;
      x[q] = i < N ? word[i] : 0;
      const uint32_t d = digit(x[q], shift, bits);
      to[q] = i < N ? base[d] + wbins[w][d] + rank[i] : 0;
      if (p == 0 && i < N && x[q] >> POS_BITS != in.none)
        reinterpret_cast<uint8_t*>(used)[x[q] >> POS_BITS] = 1;  // cleared before the barriers
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < ROUNDS; ++q)
      if (i0 + q * 64 < N) word[to[q]] = x[q];
    __syncthreads();
  }
#pragma unroll
  for (int q = 0; q < ROUNDS; ++q) {
    const int i = i0 + q * 64;
    if (i >= N) break;
    key_out[i] = word[i] >> POS_BITS;
    pos_out[i] = word[i] & (SORT_ONE - 1);
  }
}

// Chunk c of the sorted list, columns col .. col + VE - 1 per lane; `lpr` lanes per row,
// 64 / lpr chunks per wave.  A token inside the chunk is finished here; one that goes on
// from the chunk before leaves its sum in parts[c][0], one that begins here and goes on
// after it in parts[c][1].  Blocks past the chunks clear table rows without a token.
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void k_embed_sums(const uint32_t* __restrict__ key, const uint32_t* __restrict__ pos,
                                                    uint32_t none, const T* __restrict__ dout, int64_t d_stride,
                                                    float scale, T* __restrict__ dw, int64_t N, int D, int chunk,
                                                    int64_t chunks, int slices, int lpr, int64_t sum_blocks,
                                                    float* __restrict__ parts, const uint8_t* __restrict__ used,
                                                    int64_t V, int rows_per_block) {
  constexpr int VE = Vec<T>::N, U = 8;
  if (blockIdx.x >= sum_blocks) {
    const int64_t v0 = (blockIdx.x - sum_blocks) * rows_per_block;
    const int64_t v1 = v0 + rows_per_block < V ? v0 + rows_per_block : V;
    const float zero[VE] = {};
    for (int64_t v = v0 + (threadIdx.x >> 6); v < v1; v += 4)
      if (!used[v])
        for (int c = (threadIdx.x & 63) * VE; c < D; c += 64 * VE)
          store_cols<T, VE, STREAM>(dw + v * D, edge_col<VE>(c, D), D, zero);
    return;
  }
  const int64_t group = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / lpr;
  const int64_t c = group / slices;
  const int col0 = (static_cast<int>(group % slices) * lpr + threadIdx.x % lpr) * VE;
  if (c >= chunks || col0 >= D) return;
  const int col = edge_col<VE>(col0, D);
  const int64_t lo = c * chunk, hi = lo + chunk < N ? lo + chunk : N;
  uint32_t cur = key[lo];
  bool left = lo > 0 && key[lo - 1] == cur;
  float acc[VE] = {};
  const auto flush = [&](bool right) {
    if (cur == none) return;
    if (left || right) {
      float* o = parts + (c * 2 + (left ? 0 : 1)) * D + col;
      if (D >= VE) {
#pragma unroll
        for (int h = 0; h < VE / 4; ++h) {
          const float q[4] = {acc[4 * h], acc[4 * h + 1], acc[4 * h + 2], acc[4 * h + 3]};
          store_vec<4>(o + 4 * h, q);
        }
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if (col + i < D) o[i] = acc[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] *= scale;
      store_cols<T, VE, STREAM>(dw + static_cast<int64_t>(cur) * D, col, D, acc);
    }
  };
  // Rows are read one step ahead of their sums and kept packed, keys and positions two steps
  // (16 bytes each: chunks are multiples of U, and the arrays are padded).  Entries past
  // the end take row 0 and are not used; short rows (D < VE) go without the pipeline.
  static_assert(U == 8, "two 16-byte reads per step");
  u32x4 kn[2], pn[2], row[U];
  uint32_t k[U];
  const auto ids = [&](int64_t i) {
    if (i >= hi) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      kn[h] = reinterpret_cast<const u32x4*>(key + i)[h];
      pn[h] = reinterpret_cast<const u32x4*>(pos + i)[h];
    }
  };
  const auto rows = [&](int64_t i) {
    if (i >= hi) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = i + u < hi ? pn[u / 4][u % 4] : 0;
      if (D >= VE) {
        row[u] = *reinterpret_cast<const typename Vec<T>::raw*>(dout + r * d_stride + col);
      } else {
        T e[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) e[j] = dout[r * d_stride + (j < D ? j : D - 1)];
        __builtin_memcpy(&row[u], e, 16);
      }
    }
  };
  ids(lo);
  rows(lo);
  for (int64_t i = lo; i < hi; i += U) {
    float x[U][VE];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      k[u] = kn[u / 4][u % 4];
    }
    if (k[0] == none) break;  // only tokens without a gradient follow
    ids(i + U);
    u32x4 now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = row[u];
    rows(i + U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= hi) break;
      unpack<T>(now[u], x[u]);
      if (k[u] != cur) {
        flush(false);
        cur = k[u];
        left = false;
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] += x[u][e];
    }
  }
  if (cur == none) return;
  flush(hi < N && key[hi] == cur);
}

// A token that begins in chunk c and goes on: parts[c][1] + parts[c + 1][0] + ... in order,
// a quarter of them per wave, 4 columns per lane.
template <typename T>
__global__ __launch_bounds__(256) void k_embed_join(const uint32_t* __restrict__ key, uint32_t none, float scale,
                                                    T* __restrict__ dw, int64_t N, int D, int chunk, int64_t chunks,
                                                    const float* __restrict__ parts) {
  __shared__ float red[4][4][64];
  const int64_t c = blockIdx.x, lo = c * chunk, hi = lo + chunk;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, col0 = blockIdx.y * 256 + lane * 4;
  const int col = edge_col<4>(col0, D);
  if (hi >= N) return;
  const uint32_t k = key[hi], last = key[hi - 1], before = key[lo > 0 ? lo - 1 : 0];
  if (k == none || last != k || (lo > 0 && before == k)) return;
  int64_t n = 1;  // chunks c .. c + n - 1 hold the token
  for (int64_t j = c + 1 + lane;; j += 64) {
    const uint64_t m = __ballot(j < chunks && key[j * chunk] == k);
    if (m == ~uint64_t(0)) {
      n += 64;
      continue;
    }
    n += __builtin_ctzll(~m);
    break;
  }
  const int64_t q = (n + 3) / 4, a = w * q, b = a + q < n ? a + q : n;
  float s[4] = {};
  if (col0 < D) {
#pragma unroll 8
    for (int64_t j = a; j < b; ++j) {
      float x[4];
      load_cols<float, 4>(parts + ((c + j) * 2 + (j == 0 ? 1 : 0)) * D, col, D, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += x[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) red[w][i][lane] = s[i];
  __syncthreads();
  if (w != 0 || col0 >= D) return;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (col + i < D)
      from_f(dw[static_cast<int64_t>(k) * D + col + i],
             (((red[0][i][lane] + red[1][i][lane]) + red[2][i][lane]) + red[3][i][lane]) * scale);
}

// no token at all: every table row is 0
template <typename T>
__global__ __launch_bounds__(256) void k_embed_zero(T* __restrict__ dw, int64_t n) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
    from_f(dw[i], 0.f);
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

extern "C" int64_t ghm_token_logprobs_ws(int64_t rows, int64_t V, int top_k, int dtype) {
  (void)dtype;
  if (rows <= 0 || V <= 0 || top_k < 0) return 0;
  const Split p = row_split(rows, V);
  return p.parts == 1 ? 0 : rows * p.parts * (16 + 8 * static_cast<int64_t>(top_k));
}

namespace {
template <typename T, int N, int U, int W>
void launch_score(const Rows& m, int64_t rows, int V, const Ids& t, int64_t ignore, const ScoreOut& o, const Split& p,
                  void* ws, hipStream_t s) {
  constexpr int G = W == 1 ? 4 : 1;
  float4* sums = p.parts > 1 ? static_cast<float4*>(ws) : nullptr;
  uint64_t* keys = sums ? reinterpret_cast<uint64_t*>(sums + rows * p.parts) : nullptr;
  const dim3 g(static_cast<unsigned>((rows * p.parts + G - 1) / G)), b(64 * G * W);
  if (o.top_k)
    hipLaunchKernelGGL((k_score<T, N, U, W, true>), g, b, 0, s, m, rows, V, t, ignore, o, p.parts, p.len, sums, keys);
  else
    hipLaunchKernelGGL((k_score<T, N, U, W, false>), g, b, 0, s, m, rows, V, t, ignore, o, p.parts, p.len, sums, keys);
  if (sums)
    hipLaunchKernelGGL(k_score_join<T>, dim3(static_cast<unsigned>(rows)), dim3(256), 0, s, m, V, t, ignore, o, p.parts,
                       sums, keys);
}
template <typename T>
void score_any(const Rows& m, int64_t rows, int V, const Ids& t, int64_t ignore, const ScoreOut& o, void* ws,
               hipStream_t s) {
  const Split p = row_split(rows, V);
  constexpr int N = Vec<T>::N;
  if (V <= SHORT_V) {
    const dim3 g(static_cast<unsigned>((rows + 255) / 256));
    if (V <= 12) hipLaunchKernelGGL((k_score_short<T, 12>), g, dim3(256), 0, s, m, rows, V, t, ignore, o);
    else hipLaunchKernelGGL((k_score_short<T, SHORT_V>), g, dim3(256), 0, s, m, rows, V, t, ignore, o);
  } else if (V <= 64) {
    launch_score<T, 1, 1, 1>(m, rows, V, t, ignore, o, p, ws, s);
  } else if (V <= 256) {
    launch_score<T, 1, 4, 1>(m, rows, V, t, ignore, o, p, ws, s);
  } else if (V <= 64 * N) {
    launch_score<T, N, 1, 1>(m, rows, V, t, ignore, o, p, ws, s);
  } else if (V <= 128 * N) {
    launch_score<T, N, 2, 1>(m, rows, V, t, ignore, o, p, ws, s);
  } else if (one_wave(rows, V, N)) {
    launch_score<T, N, 4, 1>(m, rows, V, t, ignore, o, p, ws, s);
  } else if (o.top_k || V < 4096 * N) {
    launch_score<T, N, 4, 4>(m, rows, V, t, ignore, o, p, ws, s);
  } else {
    launch_score<T, N, 4, 8>(m, rows, V, t, ignore, o, p, ws, s);
  }
}
}  // namespace

extern "C" int ghm_token_logprobs(const void* logits, int dtype, int64_t n_inner, int64_t s_outer, int64_t s_inner,
                                  int64_t rows, int64_t V, const void* targets, int id_bits, int64_t ignore_index,
                                  int top_k, float* logprob, float* entropy, float* stats, float* top_logprob,
                                  int64_t* top_id, void* ws, int64_t ws_bytes, void* stream) {
  TOK_CHECK_ROWS();
  GHM_CHECK(top_k >= 0 && top_k <= GHM_TOP_MAX && top_k <= V, "top_k (0 .. min(64, V))");
  GHM_CHECK(!targets || ids_ok(id_bits), "id_bits (8, 32, 64)");
  GHM_CHECK(rows == 0 || (logits && (!targets || logprob) && (!logprob || targets) &&
                          (top_k == 0 || (top_logprob && top_id))), "null pointer");
  const int64_t need = ghm_token_logprobs_ws(rows, V, top_k, dtype);
  GHM_CHECK(ws_bytes >= need && (need == 0 || (ws && reinterpret_cast<uintptr_t>(ws) % 16 == 0)),
            "workspace (too small, or not 16-byte aligned)");
  if (rows == 0) return GHM_OK;
  const Rows m{logits, n_inner, s_outer, s_inner};
  const ScoreOut o{logprob, entropy, reinterpret_cast<float2*>(stats), top_logprob, top_id, top_k};
  TOK_DISPATCH(dtype, score_any<T>(m, rows, static_cast<int>(V), Ids{targets, id_bits}, ignore_index, o, ws,
                                   ghm_stream(stream)));
  return ghm_launch_status();
}

namespace {
template <typename T, int N, int U, int W>
void launch_score_bwd(const Rows& m, int64_t rows, int V, const Ids& t, int64_t ignore, const ScoreGrad& g,
                      const Split& p, T* dz, hipStream_t s) {
  constexpr int G = 4 / W;
  hipLaunchKernelGGL((k_score_bwd<T, N, U, W>), dim3(static_cast<unsigned>((rows * p.parts + G - 1) / G)), dim3(256), 0,
                     s, m, rows, V, t, ignore, g, p.parts, p.len, dz);
}
template <typename T>
void score_bwd_any(const Rows& m, int64_t rows, int V, const Ids& t, int64_t ignore, const ScoreGrad& g, void* dlogits,
                   hipStream_t s) {
  constexpr int N = Vec<T>::N;
  T* dz = static_cast<T*>(dlogits);
  const Split p = map_split(rows, V);
  if (V <= SHORT_V) {
    const dim3 gr(static_cast<unsigned>((rows + 255) / 256));
    if (V <= 12) hipLaunchKernelGGL((k_score_bwd_short<T, 12>), gr, dim3(256), 0, s, m, rows, V, t, ignore, g, dz);
    else hipLaunchKernelGGL((k_score_bwd_short<T, SHORT_V>), gr, dim3(256), 0, s, m, rows, V, t, ignore, g, dz);
  } else if (V <= 256) {
    launch_score_bwd<T, 1, 4, 1>(m, rows, V, t, ignore, g, p, dz, s);
  } else if (p.parts == 1 && one_wave(rows, V, N)) {
    launch_score_bwd<T, N, 4, 1>(m, rows, V, t, ignore, g, p, dz, s);
  } else {
    launch_score_bwd<T, N, 4, 4>(m, rows, V, t, ignore, g, p, dz, s);
  }
}
}  // namespace

extern "C" int ghm_token_logprobs_bwd(const void* logits, int dtype, int64_t n_inner, int64_t s_outer,
                                      int64_t s_inner, int64_t rows, int64_t V, const void* targets, int id_bits,
                                      int64_t ignore_index, int top_k, const int64_t* top_id, const float* stats,
                                      const float* entropy, const float* d_logprob, const float* d_entropy,
                                      const float* d_top, void* dlogits, void* stream) {
  TOK_CHECK_ROWS();
  GHM_CHECK(top_k >= 0 && top_k <= GHM_TOP_MAX && top_k <= V, "top_k (0 .. min(64, V))");
  GHM_CHECK(!targets || ids_ok(id_bits), "id_bits (8, 32, 64)");
  GHM_CHECK(rows == 0 || (logits && stats && dlogits && (!d_logprob || targets) && (!d_entropy || entropy) &&
                          (!d_top || (top_id && top_k >= 1))), "null pointer");
  if (rows == 0) return GHM_OK;
  const Rows m{logits, n_inner, s_outer, s_inner};
  const ScoreGrad g{top_id, reinterpret_cast<const float2*>(stats), entropy, d_logprob, d_entropy, d_top, top_k};
  TOK_DISPATCH(dtype, score_bwd_any<T>(m, rows, static_cast<int>(V), Ids{targets, id_bits}, ignore_index, g, dlogits,
                                       ghm_stream(stream)));
  return ghm_launch_status();
}

#define DISTILL_CHECK()                                                                                         \
  TOK_CHECK_ROWS();                                                                                             \
  GHM_CHECK(ids_ok(id_bits) && id_bits != 8 && dtype_ok(t_dtype), "top_ids (32 or 64 bits), top_logits dtype"); \
  GHM_CHECK(!targets || ids_ok(target_bits), "target_bits (8, 32, 64)");                                        \
  GHM_CHECK(k >= 1 && k <= GHM_DISTILL_MAX, "k (1 .. 1024)");                                                   \
  GHM_CHECK(temperature >= 1e-6f && temperature <= 1e6f, "temperature (1e-6 .. 1e6)");                                      \
  GHM_CHECK(alpha >= 0.f && alpha <= 1.f && (targets || alpha == 1.f), "alpha (0 .. 1; below 1 needs targets)")

namespace {
struct Distill {
  Rows m;
  int64_t rows;
  int V;
  Teacher tc;
  Ids t;
  int64_t ignore;
  Mix mix;
  float* row_loss;
  float4* stats;
  hipStream_t s;
};
// ws: counts [64] int, range sums [64] float2, then a part's sums each
constexpr int64_t DISTILL_WS_HEAD = MAX_COUNTS * 4 + MAX_COUNTS * 8;

inline Mix make_mix(bool targets, float tau, float alpha) {
  Mix x;
  x.tau = tau;
  x.it = 1.f / tau;
  x.alpha = alpha;
  x.hard = targets && alpha < 1.f;
  x.two = x.hard && alpha > 0.f && tau != 1.f;
  x.c1 = x.hard ? LOG2E : LOG2E * x.it;
  x.c2 = LOG2E * x.it;
  return x;
}

template <typename T, int N, int U, int W>
void launch_distill(const Distill& a, const Upstream& up, T* dz) {
  constexpr int G = W == 1 ? 4 : 1;
  const dim3 g(static_cast<unsigned>((a.rows + G - 1) / G)), b(64 * G * W);
  if (a.mix.two)
    hipLaunchKernelGGL((k_distill<T, N, U, W, true>), g, b, 8 * a.tc.k * G, a.s, a.m, a.rows, a.V, a.tc, a.t, a.ignore, a.mix, up,
                       a.row_loss, a.stats, dz);
  else
    hipLaunchKernelGGL((k_distill<T, N, U, W, false>), g, b, 8 * a.tc.k * G, a.s, a.m, a.rows, a.V, a.tc, a.t, a.ignore, a.mix, up,
                       a.row_loss, a.stats, dz);
}
template <typename T, int R, int W>
void launch_step(const Distill& a, const Upstream& up, T* dz) {
  constexpr int G = W == 1 ? 4 : 1;
  const dim3 g(static_cast<unsigned>((a.rows + G - 1) / G)), b(64 * G * W);
  if (a.mix.two)
    hipLaunchKernelGGL((k_distill_step<T, R, W, true>), g, b, 8 * a.tc.k * G, a.s, a.m, a.rows, a.V, a.tc, a.t, a.ignore, a.mix, up,
                       a.row_loss, a.stats, dz);
  else
    hipLaunchKernelGGL((k_distill_step<T, R, W, false>), g, b, 8 * a.tc.k * G, a.s, a.m, a.rows, a.V, a.tc, a.t, a.ignore, a.mix, up,
                       a.row_loss, a.stats, dz);
}
template <typename T, int N, int U, int W>
void launch_distill_grad(const Distill& a, const Upstream& up, const Split& p, T* dz) {
  constexpr int G = 4 / W;
  hipLaunchKernelGGL((k_distill_grad<T, N, U, W>), dim3(static_cast<unsigned>((a.rows * p.parts + G - 1) / G)), dim3(256),
                     8 * a.tc.k * G, a.s, a.m, a.rows, a.V, a.tc, a.t, a.ignore, a.mix, up, p.parts, p.len, a.stats, dz);
}
template <typename T>
void distill_short(const Distill& a, const Upstream& up, float* row_loss, T* dz) {
  const dim3 g(static_cast<unsigned>((a.rows + 255) / 256)), b(256);
  if (a.V <= 12)
    hipLaunchKernelGGL((k_distill_short<T, 12>), g, b, 0, a.s, a.m, a.rows, a.V, a.tc, a.t, a.ignore, a.mix, up,
                       row_loss, a.stats, dz);
  else
    hipLaunchKernelGGL((k_distill_short<T, SHORT_V>), g, b, 0, a.s, a.m, a.rows, a.V, a.tc, a.t, a.ignore, a.mix, up,
                       row_loss, a.stats, dz);
}
template <typename T>
void distill_grad_any(const Distill& a, const Upstream& up, T* dz) {
  constexpr int N = Vec<T>::N;
  const Split p = map_split(a.rows, a.V);
  if (a.V <= SHORT_V) distill_short<T>(a, up, nullptr, dz);
  else if (a.V <= 256) launch_distill_grad<T, 1, 4, 1>(a, up, p, dz);
  else if (p.parts == 1 && one_wave(a.rows, a.V, N)) launch_distill_grad<T, N, 4, 1>(a, up, p, dz);
  else launch_distill_grad<T, N, 4, 4>(a, up, p, dz);
}
template <typename T>
void distill_any(const Distill& a, const Upstream& up, void* dlogits, void* ws) {
  constexpr int N = Vec<T>::N;
  T* dz = static_cast<T*>(dlogits);
  const Split p = row_split(a.rows, a.V);
  const int nv = (a.V + N - 1) / N;
  if (a.V <= SHORT_V) {
    distill_short<T>(a, up, a.row_loss, dz);
  } else if (a.V <= 64) {
    launch_distill<T, 1, 1, 1>(a, up, dz);
  } else if (a.V <= 256) {
    launch_distill<T, 1, 4, 1>(a, up, dz);
  } else if (p.parts == 1 && dz && nv <= 4096) {
    if (nv <= 64) launch_step<T, 1, 1>(a, up, dz);
    else if (nv <= 128) launch_step<T, 2, 1>(a, up, dz);
    else if (nv <= 256) launch_step<T, 4, 1>(a, up, dz);
    else if (nv <= 1024) launch_step<T, 4, 4>(a, up, dz);
    else if (nv <= 2048) launch_step<T, 8, 4>(a, up, dz);
    else launch_step<T, 16, 4>(a, up, dz);
  } else if (nv <= 64) {
    launch_distill<T, N, 1, 1>(a, up, dz);
  } else if (p.parts == 1 && one_wave(a.rows, a.V, N)) {
    launch_distill<T, N, 4, 1>(a, up, dz);
  } else if (p.parts == 1 && !(dz && nv > 8192)) {
    launch_distill<T, N, 4, 8>(a, up, dz);
  } else if (p.parts == 1) {
    launch_distill<T, N, 4, 16>(a, up, dz);
  } else {
    float4* sums = reinterpret_cast<float4*>(static_cast<char*>(ws) + DISTILL_WS_HEAD);
    const dim3 g(static_cast<unsigned>(a.rows * p.parts)), g1(static_cast<unsigned>(a.rows));
    if (a.mix.two) {
      hipLaunchKernelGGL((k_distill_part<T, N, 4, 8, true>), g, dim3(512), 0, a.s, a.m, a.V, a.tc, a.t, a.ignore, a.mix,
                         p.parts, p.len, sums);
      hipLaunchKernelGGL((k_distill_join<T, true>), g1, dim3(256), 8 * a.tc.k, a.s, a.m, a.V, a.tc, a.t, a.ignore, a.mix, p.parts,
                         sums, a.row_loss, a.stats);
    } else {
      hipLaunchKernelGGL((k_distill_part<T, N, 4, 8, false>), g, dim3(512), 0, a.s, a.m, a.V, a.tc, a.t, a.ignore, a.mix,
                         p.parts, p.len, sums);
      hipLaunchKernelGGL((k_distill_join<T, false>), g1, dim3(256), 8 * a.tc.k, a.s, a.m, a.V, a.tc, a.t, a.ignore, a.mix, p.parts,
                         sums, a.row_loss, a.stats);
    }
    if (dz) distill_grad_any<T>(a, up, dz);
  }
}
}  // namespace

extern "C" int64_t ghm_distill_ws(int64_t rows, int64_t V, int dtype) {
  (void)dtype;
  if (rows <= 0 || V <= 0) return DISTILL_WS_HEAD;
  const Split p = row_split(rows, V);
  return DISTILL_WS_HEAD + (p.parts == 1 ? 0 : rows * p.parts * 16);
}

extern "C" int ghm_distill(const void* logits, int dtype, int64_t n_inner, int64_t s_outer, int64_t s_inner,
                           int64_t rows, int64_t V, const void* top_ids, int id_bits, const void* top_logits,
                           int t_dtype, int k, const void* targets, int target_bits, int64_t ignore_index,
                           float temperature, float alpha, int reduction, float* loss, float* row_loss, float* stats,
                           float* norm, float grad_scale, void* dlogits, void* ws, int64_t ws_bytes, void* stream) {
  DISTILL_CHECK();
  GHM_CHECK(reduction >= 0 && reduction <= 2, "reduction (0 none, 1 mean, 2 sum)");
  GHM_CHECK((reduction == 0 || loss) && (reduction != 1 || norm), "null pointer");
  GHM_CHECK(rows == 0 || (logits && top_ids && top_logits && row_loss && stats), "null pointer");
  GHM_CHECK(reinterpret_cast<uintptr_t>(stats) % 16 == 0, "stats (16-byte aligned)");
  GHM_CHECK(ws && ws_bytes >= ghm_distill_ws(rows, V, dtype) && reinterpret_cast<uintptr_t>(ws) % 16 == 0,
            "workspace (too small, or not 16-byte aligned)");
  const Distill a{{logits, n_inner, s_outer, s_inner}, rows, static_cast<int>(V), {{top_ids, id_bits}, top_logits, t_dtype, k},
                  {targets, target_bits}, ignore_index, make_mix(targets != nullptr, temperature, alpha), row_loss,
                  reinterpret_cast<float4*>(stats), ghm_stream(stream)};
  int* counts = static_cast<int*>(ws);
  float2* ranges = reinterpret_cast<float2*>(counts + MAX_COUNTS);
  Upstream up{nullptr, 0, nullptr, nullptr, 0, grad_scale};
  if (rows && dlogits && reduction == 1) {  // the gradient needs the number of counted rows first
    const int nb = static_cast<int>((rows + 255) / 256 < MAX_COUNTS ? (rows + 255) / 256 : MAX_COUNTS);
    hipLaunchKernelGGL(k_distill_count, dim3(nb), dim3(256), 0, a.s, a.tc, a.t, ignore_index, rows, (rows + nb - 1) / nb,
                       counts);
    up.counts = counts;
    up.n_counts = nb;
  }
  if (rows) TOK_DISPATCH(dtype, distill_any<T>(a, up, dlogits, ws));
  if (reduction) {
    // one block up to 16,384 rows, ranges of that many (at most 64) above
    const int nb = static_cast<int>((rows + 16383) / 16384 < 1 ? 1 : (rows + 16383) / 16384 < MAX_COUNTS ? (rows + 16383) / 16384 : MAX_COUNTS);
    hipLaunchKernelGGL(k_distill_total, dim3(nb), dim3(1024), 0, a.s, row_loss, a.stats, rows, (rows + nb - 1) / nb,
                       ranges, reduction == 1, loss, norm);
    if (nb > 1)
      hipLaunchKernelGGL(k_distill_total2, dim3(1), dim3(64), 0, a.s, ranges, nb, reduction == 1, loss, norm);
  }
  return ghm_launch_status();
}

extern "C" int ghm_distill_bwd(const void* logits, int dtype, int64_t n_inner, int64_t s_outer, int64_t s_inner,
                               int64_t rows, int64_t V, const void* top_ids, int id_bits, const void* top_logits,
                               int t_dtype, int k, const void* targets, int target_bits, int64_t ignore_index,
                               float temperature, float alpha, const float* stats, const float* norm,
                               const float* d_loss, int d_rows, void* dlogits, void* stream) {
  DISTILL_CHECK();
  GHM_CHECK(rows == 0 || (logits && top_ids && top_logits && stats && d_loss && dlogits), "null pointer");
  GHM_CHECK(reinterpret_cast<uintptr_t>(stats) % 16 == 0, "stats (16-byte aligned)");
  if (rows == 0) return GHM_OK;
  const Distill a{{logits, n_inner, s_outer, s_inner}, rows, static_cast<int>(V), {{top_ids, id_bits}, top_logits, t_dtype, k},
                  {targets, target_bits}, ignore_index, make_mix(targets != nullptr, temperature, alpha), nullptr,
                  reinterpret_cast<float4*>(const_cast<float*>(stats)), ghm_stream(stream)};
  const Upstream up{nullptr, 0, norm, d_loss, d_rows, 1.f};
  TOK_DISPATCH(dtype, distill_grad_any<T>(a, up, static_cast<T*>(dlogits)));
  return ghm_launch_status();
}

#define EMBED_CHECK()                                                                                              \
  GHM_CHECK(dtype_ok(dtype) && ids_ok(id_bits), "dtype (0 f32, 1 bf16, 2 f16), id_bits (8, 32, 64)");              \
  GHM_CHECK(N >= 0 && N < (int64_t(1) << 31) && V >= 1 && V < (int64_t(1) << 31) && D >= 1 && D <= (int64_t(1) << 20), \
            "shape (N, V < 2^31, D <= 2^20)")

namespace {
// rows of whole 64-byte lines are stored past the caches: the gradient of 16,384 x 2048
// bf16 tokens into 65,536 rows took 98 us that way and 114 us through them; rows that share
// lines (1001 f32 values) 164 us and 163 us
inline bool whole_lines(const void* p, int64_t row_bytes) {
  return reinterpret_cast<uintptr_t>(p) % 64 == 0 && row_bytes % 64 == 0;
}
}  // namespace

extern "C" int ghm_embed_rows_fwd(const void* tokens, int id_bits, const void* weight, int dtype, int64_t w_stride,
                                  float scale, void* out, int64_t N, int64_t V, int64_t D, void* stream) {
  EMBED_CHECK();
  GHM_CHECK(w_stride >= 0, "row stride");
  GHM_CHECK(N == 0 || (tokens && weight && out), "null pointer");
  if (N == 0) return GHM_OK;
  const int ve = dtype == 0 ? 4 : 8, vecs = static_cast<int>((D + ve - 1) / ve);
  const int per = vecs >= 1024 ? 1 : 1024 / vecs;
  const dim3 g(static_cast<unsigned>((N + per - 1) / per)), b(256);
  const Ids t{tokens, id_bits};
  const int d = static_cast<int>(D);
  hipStream_t s = ghm_stream(stream);
  if (whole_lines(out, D * (16 / ve)))
    TOK_DISPATCH(dtype, hipLaunchKernelGGL((k_embed_rows<T, true>), g, b, 0, s, t, static_cast<const T*>(weight), w_stride,
                                           scale, static_cast<T*>(out), N, V, d, vecs, per));
  else
    TOK_DISPATCH(dtype, hipLaunchKernelGGL((k_embed_rows<T, false>), g, b, 0, s, t, static_cast<const T*>(weight),
                                           w_stride, scale, static_cast<T*>(out), N, V, d, vecs, per));
  return ghm_launch_status();
}

namespace {
struct EmbedPlan {
  int passes, bits, chunk, slices, lpr;
  int64_t chunks, used_words;
  int64_t key[2], pos[2], counts, used, parts, bytes;  // byte offsets in the workspace
};
inline int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
inline EmbedPlan embed_plan(int64_t N, int64_t V, int64_t D, int ve) {
  EmbedPlan p;
  int bits = 1;
  while (bits < 32 && (int64_t(1) << bits) <= V) ++bits;  // keys 0 .. V
  p.passes = (bits + SORT_BITS - 1) / SORT_BITS;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.lpr = 1;
  while (p.lpr < 64 && p.lpr * ve < D) p.lpr *= 2;
  p.slices = static_cast<int>((D + p.lpr * ve - 1) / (p.lpr * ve));
  const int64_t want = N * p.slices / (2048 * (64 / p.lpr));
  p.chunk = 16;
  while (p.chunk < 256 && p.chunk < want) p.chunk *= 2;
  p.chunks = (N + p.chunk - 1) / p.chunk;
  p.used_words = (V + 3) / 4;
  int64_t at = 0;
  for (int i = 0; i < 2; ++i) {
    p.key[i] = at, at += up256(N * 4);
    p.pos[i] = at, at += up256(N * 4);
  }
  p.counts = at, at += up256((N / (64 * 4 * SORT_ROUNDS) + 2) * SORT_BINS * 4);
  p.used = at, at += up256(p.used_words * 4);
  p.parts = at, at += up256(p.chunks * 2 * D * 4);
  p.bytes = at;
  return p;
}

template <int W, int MODE>
void launch_sort(const EmbedPlan& p, const Ids& tok, int64_t pad, int64_t N, int64_t V, char* ws, hipStream_t s) {
  uint32_t* counts = reinterpret_cast<uint32_t*>(ws + p.counts);
  uint32_t* used = reinterpret_cast<uint32_t*>(ws + p.used);
  const int64_t tile = 64 * W * SORT_ROUNDS, tiles = (N + tile - 1) / tile;
  const dim3 g(static_cast<unsigned>(tiles)), b(64 * W);
  for (int i = 0; i < p.passes; ++i) {
    SortIn in{tok, nullptr, nullptr, pad, static_cast<uint32_t>(V)};
    if (i > 0) {
      in.key = reinterpret_cast<uint32_t*>(ws + p.key[(i - 1) & 1]);
      in.pos = reinterpret_cast<uint32_t*>(ws + p.pos[(i - 1) & 1]);
    }
    if (MODE != SORT_SELF)
      hipLaunchKernelGGL(k_sort_count<W>, g, b, 0, s, in, N, i * p.bits, p.bits, counts, i == 0 ? used : nullptr, p.used_words);
    if (MODE == SORT_SCANNED) hipLaunchKernelGGL(k_sort_scan, dim3(SORT_BINS / 64), dim3(64), 0, s, counts, tiles);
    // cleared by the first launch, set by the second; a single one writes every row's from its counts
    const bool one_pass = MODE == SORT_SELF && p.passes == 1, clear = MODE == SORT_SELF && i == 0 && !one_pass;
    const bool set = MODE == SORT_SELF ? one_pass || i == 1 : i == 0;
    hipLaunchKernelGGL((k_sort_scatter<W, MODE>), g, b, 0, s, in, N, i * p.bits, p.bits, counts, static_cast<int>(tiles),
                       reinterpret_cast<uint32_t*>(ws + p.key[i & 1]), reinterpret_cast<uint32_t*>(ws + p.pos[i & 1]),
                       set ? reinterpret_cast<uint8_t*>(used) : nullptr, one_pass, clear ? used : nullptr, p.used_words);
  }
}
template <typename T>
void embed_bwd_any(const Ids& tok, const T* dout, int64_t d_stride, float scale, int64_t pad, T* dw, int64_t N, int64_t V,
                   int D, char* ws, hipStream_t s) {
  if (N == 0) {
    const int64_t n = V * D, blocks = (n + 1023) / 1024;
    hipLaunchKernelGGL(k_embed_zero<T>, dim3(static_cast<unsigned>(blocks < 8192 ? blocks : 8192)), dim3(256), 0, s, dw, n);
    return;
  }
  const EmbedPlan p = embed_plan(N, V, D, Vec<T>::N);
  uint32_t* key = reinterpret_cast<uint32_t*>(ws + p.key[(p.passes - 1) & 1]);
  uint32_t* pos = reinterpret_cast<uint32_t*>(ws + p.pos[(p.passes - 1) & 1]);
  if (N <= SORT_ONE && V <= USED_ONE) {
    const SortIn in{tok, nullptr, nullptr, pad, static_cast<uint32_t>(V)};
    hipLaunchKernelGGL(k_sort_one, dim3(1), dim3(1024), 0, s, in, static_cast<int>(N), p.passes, p.bits, key, pos,
                       reinterpret_cast<uint32_t*>(ws + p.used), static_cast<int>(p.used_words));
  } else if (N <= SORT_SELF_N) {
    launch_sort<8, SORT_SELF>(p, tok, pad, N, V, ws, s);
  } else if (N <= 64 * 4 * SORT_ROUNDS * SORT_TILES) {
    launch_sort<4, SORT_SUM>(p, tok, pad, N, V, ws, s);
  } else {
    launch_sort<16, SORT_SCANNED>(p, tok, pad, N, V, ws, s);
  }
  float* parts = reinterpret_cast<float*>(ws + p.parts);
  const uint8_t* used = reinterpret_cast<uint8_t*>(ws + p.used);
  const int64_t sum_blocks = (p.chunks * p.slices * p.lpr + 255) / 256;
  // about 64 KiB of table rows per clearing block, at most 2^20 of them
  int64_t rpb = 65536 / (D * static_cast<int64_t>(sizeof(T)));
  if (rpb < 4) rpb = 4;
  if (rpb > 4096) rpb = 4096;
  while ((V + rpb - 1) / rpb > (1 << 20)) rpb *= 2;
  const int64_t zero_blocks = (V + rpb - 1) / rpb;
  const dim3 g(static_cast<unsigned>(sum_blocks + zero_blocks)), b(256);
  const uint32_t none = static_cast<uint32_t>(V);
  if (whole_lines(dw, D * static_cast<int64_t>(sizeof(T))))
    hipLaunchKernelGGL((k_embed_sums<T, true>), g, b, 0, s, key, pos, none, dout, d_stride, scale, dw, N, D, p.chunk,
                       p.chunks, p.slices, p.lpr, sum_blocks, parts, used, V, static_cast<int>(rpb));
  else
    hipLaunchKernelGGL((k_embed_sums<T, false>), g, b, 0, s, key, pos, none, dout, d_stride, scale, dw, N, D, p.chunk,
                       p.chunks, p.slices, p.lpr, sum_blocks, parts, used, V, static_cast<int>(rpb));
  if (p.chunks > 1)
    hipLaunchKernelGGL(k_embed_join<T>, dim3(static_cast<unsigned>(p.chunks - 1), static_cast<unsigned>((D + 255) / 256)),
                       dim3(256), 0, s, key, static_cast<uint32_t>(V), scale, dw, N, D, p.chunk, p.chunks, parts);
}
}  // namespace

extern "C" int64_t ghm_embed_rows_bwd_ws(int64_t N, int64_t V, int64_t D) {
  if (N <= 0 || V <= 0 || D <= 0) return 0;
  const int64_t a = embed_plan(N, V, D, 4).bytes, b = embed_plan(N, V, D, 8).bytes;
  return a > b ? a : b;
}

extern "C" int ghm_embed_rows_bwd(const void* tokens, int id_bits, const void* dout, int dtype, int64_t d_stride,
                                  float scale, int64_t padding_idx, void* dweight, int64_t N, int64_t V, int64_t D,
                                  void* ws, int64_t ws_bytes, void* stream) {
  EMBED_CHECK();
  GHM_CHECK(d_stride >= 0 && padding_idx >= -1 && padding_idx < V, "row stride, padding_idx (-1 .. V - 1)");
  GHM_CHECK(dweight && (N == 0 || (tokens && dout)), "null pointer");
  const int64_t need = ghm_embed_rows_bwd_ws(N, V, D);
  GHM_CHECK(ws_bytes >= need && (need == 0 || (ws && reinterpret_cast<uintptr_t>(ws) % 16 == 0)),
            "workspace (too small, or not 16-byte aligned)");
  TOK_DISPATCH(dtype, embed_bwd_any<T>(Ids{tokens, id_bits}, static_cast<const T*>(dout), d_stride, scale, padding_idx,
                                       static_cast<T*>(dweight), N, V, static_cast<int>(D), static_cast<char*>(ws),
                                       ghm_stream(stream)));
  return ghm_launch_status();
}
