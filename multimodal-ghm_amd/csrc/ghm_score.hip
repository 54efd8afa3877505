// Log probabilities of given tokens under softmax(logits), with the entropy and the most
// likely values of each row, from one pass over the logits; and their gradient.
#include "ghm_token.h"

namespace {

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
  uint64_t last = 0;  // a NaN of id 0 has the largest key there is: the first search has no bound
  for (int j = 0; j < k; ++j) {
    uint64_t best = 0;
    for (int v = lo + w * 64 + lane; v < hi; v += W * 64) {
      const uint64_t key = top_key(to_f(z[v]), v);
      best = (j == 0 || key < last) && key > best ? key : best;
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

// One pass: every value is read once, with the running maximum, the two sums and the noting
// of vectors on the vector unit meanwhile (about 11 instructions a value, the exponential
// counting four).  Bound by the reads: 4,096 rows of 131,072 bf16 values in 182 us (5.9 TB/s;
// a copy of 2 GiB runs at 4.9), with the 32 most likely values 219 us; 2,000 rows of 50,001
// f32 values 70 us (5.8 TB/s).  Four waves per row leave more rows in flight beside one that
// ranks its alternatives (eight: 230 us); without alternatives eight are 5 % faster.
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
  const int64_t item = block_number() * G + wave / W;
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
template <typename T, int M>
__global__ __launch_bounds__(64) void k_score_short(Rows rows, int64_t n_rows, int V, Ids targets, int64_t ignore,
                                                    ScoreOut out) {
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x;
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

// The whole row part is written first, then the target's and the alternatives' entries again.
// Bound by one read and one write.  The last rows come first, and the stores go past the caches:
// what the scores read last is still in the 256 MB one where the gradient follows at once.  Scores
// and gradient of 2,000 rows of 50,001 f32 values 205 us (251 in order and through the caches),
// of 4,096 x 32,000 bf16 135 (165); the gradient alone 157 (5.1 TB/s).
template <typename T, int N, int U, int W>
__global__ __launch_bounds__(256) void k_score_bwd(Rows rows, int64_t n_rows, int V, Ids targets, int64_t ignore,
                                                   ScoreGrad g, int parts, int part_len, T* __restrict__ dz) {
  constexpr int G = 4 / W;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, w = wave % W;
  const int64_t item = n_rows * parts - 1 - (block_number() * G + wave / W);
  if (item < 0) return;
  const int64_t r = item / parts;
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
  map_row<T, N, U, W, true, true>(z, d, lo, hi, w, lane, f);
  group_sync<W>();
  if (w != 0) return;
  const int64_t id = g.g_top && lane < g.top_k ? g.top_id[r * g.top_k + lane] : -1;
  if (id >= lo && id < hi)
    from_f(d[id], f(to_f(z[id])) + g.g_top[r * g.top_k + lane] + (g.g_lp && id == y ? g1 : 0.f));
  if (g.g_lp && y >= lo && y < hi && __ballot(id == y) == 0 && lane == 0) from_f(d[y], f(to_f(z[y])) + g1);
}

template <typename T, int M>
__global__ __launch_bounds__(64) void k_score_bwd_short(Rows rows, int64_t n_rows, int V, Ids targets, int64_t ignore,
                                                        ScoreGrad g, T* __restrict__ dz) {
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x;
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

}  // namespace

extern "C" int64_t ghm_token_logprobs_ws(int64_t rows, int64_t V, int top_k, int dtype) {
  if (rows <= 0 || V <= 0 || top_k < 0) return 0;
  const Split p = row_split(rows, V, dtype == 0 ? 4 : 8, top_k ? SPLIT_TOP : SPLIT_SUMS);
  return p.parts == 1 ? 0 : rows * p.parts * (16 + 8 * static_cast<int64_t>(top_k));
}

namespace {
template <typename T, int N, int U, int W>
void launch_score(const Rows& m, int64_t rows, int V, const Ids& t, int64_t ignore, const ScoreOut& o, const Split& p,
                  void* ws, hipStream_t s) {
  constexpr int G = W == 1 ? 4 : 1;
  float4* sums = p.parts > 1 ? static_cast<float4*>(ws) : nullptr;
  uint64_t* keys = sums ? reinterpret_cast<uint64_t*>(sums + rows * p.parts) : nullptr;
  const dim3 g = grid_of((rows * p.parts + G - 1) / G, 64 * G * W), b(64 * G * W);
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
  constexpr int N = Vec<T>::N;
  const Split p = row_split(rows, V, N, o.top_k ? SPLIT_TOP : SPLIT_SUMS);
  if (V <= SHORT_V) {
    const dim3 g(static_cast<unsigned>((rows + 63) / 64));
    if (V <= 12) hipLaunchKernelGGL((k_score_short<T, 12>), g, dim3(64), 0, s, m, rows, V, t, ignore, o);
    else hipLaunchKernelGGL((k_score_short<T, SHORT_V>), g, dim3(64), 0, s, m, rows, V, t, ignore, o);
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
  hipLaunchKernelGGL((k_score_bwd<T, N, U, W>), grid_of((rows * p.parts + G - 1) / G, 256), dim3(256), 0, s, m, rows, V, t,
                     ignore, g, p.parts, p.len, dz);
}
template <typename T>
void score_bwd_any(const Rows& m, int64_t rows, int V, const Ids& t, int64_t ignore, const ScoreGrad& g, void* dlogits,
                   hipStream_t s) {
  constexpr int N = Vec<T>::N;
  T* dz = static_cast<T*>(dlogits);
  const Split p = map_split(rows, V);
  if (V <= SHORT_V) {
    const dim3 gr(static_cast<unsigned>((rows + 63) / 64));
    if (V <= 12) hipLaunchKernelGGL((k_score_bwd_short<T, 12>), gr, dim3(64), 0, s, m, rows, V, t, ignore, g, dz);
    else hipLaunchKernelGGL((k_score_bwd_short<T, SHORT_V>), gr, dim3(64), 0, s, m, rows, V, t, ignore, g, dz);
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
