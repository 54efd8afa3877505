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

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float NEG_INF = -__builtin_inff();
constexpr int TOK_THREADS = 256;

struct bf16_t { uint16_t u; };
struct f16_t { _Float16 h; };

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(bf16_t x) { return __uint_as_float(static_cast<uint32_t>(x.u) << 16); }
__device__ __forceinline__ float to_f(f16_t x) { return static_cast<float>(x.h); }
__device__ __forceinline__ void from_f(float& o, float x) { o = x; }
__device__ __forceinline__ void from_f(bf16_t& o, float x) { o.u = __builtin_bit_cast(uint16_t, static_cast<__bf16>(x)); }
__device__ __forceinline__ void from_f(f16_t& o, float x) { o.h = static_cast<_Float16>(x); }

// e^x from the exponent's own 32-bit unit: 2^(x log2 e), 0 below the f32 range
__device__ __forceinline__ float exp_f(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

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

template <typename F>
__device__ __forceinline__ float block_reduce(float v, float* red, F f) {
  __syncthreads();
  red[threadIdx.x] = v;
  __syncthreads();
  for (int s = TOK_THREADS / 2; s >= 1; s >>= 1) {
    if (threadIdx.x < s) red[threadIdx.x] = f(red[threadIdx.x], red[threadIdx.x + s]);
    __syncthreads();
  }
  return red[0];
}
__device__ __forceinline__ float block_max(float v, float* red) {
  return block_reduce(v, red, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float block_sum(float v, float* red) {
  return block_reduce(v, red, [](float a, float b) { return a + b; });
}

// ---------------------------------------------------------------------------
// Scores: m = max z, s = sum e^(z - m), log p_v = (z_v - m) - log s,
// H = log s - sum e^(z - m) (z - m) / s.  A value of -inf has probability 0 and
// adds nothing; a row without a finite maximum has no distribution (NaN).
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(TOK_THREADS) void k_score(Rows rows, int V, Ids targets, int64_t ignore, int top_k,
                                                       float* __restrict__ logprob, float* __restrict__ entropy,
                                                       float2* __restrict__ stats, float* __restrict__ top_lp,
                                                       int64_t* __restrict__ top_id) {
  __shared__ float red[TOK_THREADS];
  __shared__ uint64_t kred[TOK_THREADS];
  const int64_t r = blockIdx.x;
  const int64_t y = targets.p ? ld_id(targets, r) : 0;
  if (targets.p && y == ignore) {  // padding: nothing of the row is read
    if (threadIdx.x == 0) {
      logprob[r] = 0.f;
      if (entropy) entropy[r] = 0.f;
      if (stats) stats[r] = make_float2(0.f, 0.f);
    }
    for (int j = threadIdx.x; j < top_k; j += TOK_THREADS) {
      top_lp[r * top_k + j] = 0.f;
      top_id[r * top_k + j] = -1;
    }
    return;
  }
  const T* z = row_ptr<T>(rows, r);
  float m = -FLT_MAX;
  for (int v = threadIdx.x; v < V; v += TOK_THREADS) m = fmaxf(m, to_f(z[v]));
  m = block_max(m, red);
  float s = 0.f, t = 0.f;
  for (int v = threadIdx.x; v < V; v += TOK_THREADS) {
    const float d = to_f(z[v]) - m, e = exp_f(d);
    s += e;
    t += e * fmaxf(d, -1e4f);
  }
  s = block_sum(s, red);
  t = block_sum(t, red);
  const float ls = logf(s);
  if (threadIdx.x == 0) {
    if (logprob) logprob[r] = y >= 0 && y < V ? (to_f(z[y]) - m) - ls : __builtin_nanf("");
    if (entropy) entropy[r] = ls - t / s;
    if (stats) stats[r] = make_float2(m, ls);
  }
  uint64_t last = ~0ull;
  for (int j = 0; j < top_k; ++j) {
    uint64_t best = 0;
    for (int v = threadIdx.x; v < V; v += TOK_THREADS) {
      const uint64_t k = top_key(to_f(z[v]), v);
      if (k < last && k > best) best = k;
    }
    __syncthreads();
    kred[threadIdx.x] = best;
    __syncthreads();
    for (int w = TOK_THREADS / 2; w >= 1; w >>= 1) {
      if (threadIdx.x < w && kred[threadIdx.x + w] > kred[threadIdx.x]) kred[threadIdx.x] = kred[threadIdx.x + w];
      __syncthreads();
    }
    last = kred[0];
    if (threadIdx.x == 0) {
      const uint32_t v = 0xffffffffu - static_cast<uint32_t>(last);
      top_id[r * top_k + j] = v;
      top_lp[r * top_k + j] = (to_f(z[v]) - m) - ls;
    }
  }
}

// dz_v = -p_v [g_lp + sum_j g_top_j + g_H (log p_v + H)] + g_lp [v = y] + sum_j g_top_j [v = id_j]
template <typename T>
__global__ __launch_bounds__(TOK_THREADS) void k_score_bwd(Rows rows, int V, Ids targets, int64_t ignore, int top_k,
                                                           const int64_t* __restrict__ top_id,
                                                           const float2* __restrict__ stats,
                                                           const float* __restrict__ entropy,
                                                           const float* __restrict__ g_lp,
                                                           const float* __restrict__ g_ent,
                                                           const float* __restrict__ g_top, T* __restrict__ dz) {
  const int64_t r = blockIdx.x;
  T* d = dz + r * V;
  const int64_t y = targets.p ? ld_id(targets, r) : 0;
  if (targets.p && y == ignore) {
    for (int v = threadIdx.x; v < V; v += TOK_THREADS) from_f(d[v], 0.f);
    return;
  }
  const T* z = row_ptr<T>(rows, r);
  const float2 st = stats[r];
  float g1 = g_lp ? g_lp[r] : 0.f;
  if (g_lp && (y < 0 || y >= V)) g1 = __builtin_nanf("");
  const float g2 = g_ent ? g_ent[r] : 0.f, H = g_ent ? entropy[r] : 0.f;
  float gs = g1;
  for (int j = 0; j < top_k; ++j) gs += g_top[r * top_k + j];
  for (int v = threadIdx.x; v < V; v += TOK_THREADS) {
    const float lp = (to_f(z[v]) - st.x) - st.y, p = exp_f(lp);
    float g = -p * (gs + g2 * (fmaxf(lp, -1e4f) + H));
    if (g_lp && v == y) g += g1;
    for (int j = 0; j < top_k; ++j)
      if (top_id[r * top_k + j] == v) g += g_top[r * top_k + j];
    from_f(d[v], g);
  }
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
// rows that count: the target is not the ignored one; without targets, an alternative is present
__device__ __forceinline__ bool row_counts(const Teacher& t, const Ids& targets, int64_t ignore, int64_t r) {
  if (targets.p) return ld_id(targets, r) != ignore;
  for (int j = 0; j < t.k; ++j)
    if (teacher_has(t, r * t.k + j)) return true;
  return false;
}

// norm[0] = 1 / max(number of counted rows, 1)
__global__ __launch_bounds__(TOK_THREADS) void k_distill_count(Teacher t, Ids targets, int64_t ignore, int64_t n,
                                                               float* __restrict__ norm) {
  __shared__ int red[TOK_THREADS];
  int c = 0;
  for (int64_t r = threadIdx.x; r < n; r += TOK_THREADS) c += row_counts(t, targets, ignore, r);
  red[threadIdx.x] = c;
  __syncthreads();
  for (int s = TOK_THREADS / 2; s >= 1; s >>= 1) {
    if (threadIdx.x < s) red[threadIdx.x] += red[threadIdx.x + s];
    __syncthreads();
  }
  if (threadIdx.x == 0) norm[0] = 1.f / static_cast<float>(red[0] > 1 ? red[0] : 1);
}

// row_stats: (m, log s at 1, log s at tau, unused)
template <typename T>
__global__ __launch_bounds__(TOK_THREADS) void k_distill_rows(Rows rows, int V, Teacher tc, Ids targets,
                                                              int64_t ignore, float tau, float alpha,
                                                              float* __restrict__ row_loss,
                                                              float4* __restrict__ row_stats) {
  __shared__ float red[TOK_THREADS];
  const int64_t r = blockIdx.x;
  if (!row_counts(tc, targets, ignore, r)) {
    if (threadIdx.x == 0) {
      row_loss[r] = 0.f;
      row_stats[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    return;
  }
  const T* z = row_ptr<T>(rows, r);
  const float it = 1.f / tau;
  float m = -FLT_MAX;
  for (int v = threadIdx.x; v < V; v += TOK_THREADS) m = fmaxf(m, to_f(z[v]));
  m = block_max(m, red);
  float s1 = 0.f, s2 = 0.f;
  for (int v = threadIdx.x; v < V; v += TOK_THREADS) {
    const float d = to_f(z[v]) - m;
    s1 += exp_f(d);
    s2 += exp_f(d * it);
  }
  const float l1 = logf(block_sum(s1, red)), l2 = logf(block_sum(s2, red));
  float mt = -FLT_MAX;
  for (int j = threadIdx.x; j < tc.k; j += TOK_THREADS)
    if (teacher_has(tc, r * tc.k + j)) mt = fmaxf(mt, ld_teacher(tc, r * tc.k + j));
  mt = block_max(mt, red);
  float st = 0.f;
  for (int j = threadIdx.x; j < tc.k; j += TOK_THREADS)
    if (teacher_has(tc, r * tc.k + j)) st += exp_f((ld_teacher(tc, r * tc.k + j) - mt) * it);
  st = block_sum(st, red);
  const float lt = logf(st);
  float kl = 0.f;
  for (int j = threadIdx.x; j < tc.k; j += TOK_THREADS) {
    if (!teacher_has(tc, r * tc.k + j)) continue;
    const int64_t v = ld_id(tc.ids, r * tc.k + j);
    const float lq = (ld_teacher(tc, r * tc.k + j) - mt) * it - lt, q = exp_f(lq);
    if (v >= V) kl = __builtin_nanf("");
    else if (!(q == 0.f)) kl += q * (lq - ((to_f(z[v]) - m) * it - l2));
  }
  kl = block_sum(kl, red);
  if (threadIdx.x == 0) {
    float loss = alpha * tau * tau * kl;
    if (targets.p) {
      const int64_t y = ld_id(targets, r);
      loss += (1.f - alpha) * (y >= 0 && y < V ? l1 - (to_f(z[y]) - m) : __builtin_nanf(""));
    }
    row_loss[r] = loss;
    row_stats[r] = make_float4(m, l1, l2, 0.f);
  }
}

// the gradient of one row: scale = grad_scale * upstream * norm
template <typename T>
__global__ __launch_bounds__(TOK_THREADS) void k_distill_grad(Rows rows, int V, Teacher tc, Ids targets,
                                                              int64_t ignore, float tau, float alpha,
                                                              const float4* __restrict__ row_stats,
                                                              const float* __restrict__ norm,
                                                              const float* __restrict__ up, int up_rows,
                                                              float grad_scale, T* __restrict__ dz) {
  __shared__ float red[TOK_THREADS];
  const int64_t r = blockIdx.x;
  T* d = dz + r * V;
  if (!row_counts(tc, targets, ignore, r)) {
    for (int v = threadIdx.x; v < V; v += TOK_THREADS) from_f(d[v], 0.f);
    return;
  }
  const T* z = row_ptr<T>(rows, r);
  float scale = grad_scale;
  if (norm) scale *= norm[0];
  if (up) scale *= up[up_rows ? r : 0];
  const float4 st = row_stats[r];
  const float it = 1.f / tau;
  float mt = -FLT_MAX;
  for (int j = threadIdx.x; j < tc.k; j += TOK_THREADS)
    if (teacher_has(tc, r * tc.k + j)) mt = fmaxf(mt, ld_teacher(tc, r * tc.k + j));
  mt = block_max(mt, red);
  float s = 0.f, bad = 0.f;
  for (int j = threadIdx.x; j < tc.k; j += TOK_THREADS)
    if (teacher_has(tc, r * tc.k + j)) {
      s += exp_f((ld_teacher(tc, r * tc.k + j) - mt) * it);
      if (ld_id(tc.ids, r * tc.k + j) >= V) bad = 1.f;
    }
  s = block_sum(s, red);
  bad = block_max(bad, red);
  const float lt = logf(s);
  const float has = s == 0.f ? 0.f : 1.f;
  const int64_t y = targets.p ? ld_id(targets, r) : -1;
  if (bad != 0.f || (targets.p && (y < 0 || y >= V))) scale = __builtin_nanf("");
  for (int v = threadIdx.x; v < V; v += TOK_THREADS) {
    const float dv = to_f(z[v]) - st.x;
    float soft = has != 0.f ? exp_f(dv * it - st.z) : 0.f;
    for (int j = 0; j < tc.k; ++j)
      if (ld_id(tc.ids, r * tc.k + j) == v && teacher_has(tc, r * tc.k + j))
        soft -= exp_f((ld_teacher(tc, r * tc.k + j) - mt) * it - lt);
    float g = alpha * tau * soft;
    if (targets.p) g += (1.f - alpha) * (exp_f(dv - st.y) - (v == y ? 1.f : 0.f));
    from_f(d[v], scale * g);
  }
}

// loss[0] = norm * sum of row losses (norm NULL: the sum), one fixed order
__global__ __launch_bounds__(TOK_THREADS) void k_distill_total(const float* __restrict__ row_loss, int64_t n,
                                                               const float* __restrict__ norm,
                                                               float* __restrict__ loss) {
  __shared__ float red[TOK_THREADS];
  float s = 0.f;
  for (int64_t r = threadIdx.x; r < n; r += TOK_THREADS) s += row_loss[r];
  s = block_sum(s, red);
  if (threadIdx.x == 0) loss[0] = norm ? s * norm[0] : s;
}

// ---------------------------------------------------------------------------
// Scaled embedding: out_i = scale W[tok_i]; dW_v = scale sum_{i: tok_i = v} dout_i,
// summed in f32 in ascending i and rounded once.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(TOK_THREADS) void k_embed_rows(Ids tok, const T* __restrict__ w, int64_t w_stride,
                                                            float scale, T* __restrict__ out, int64_t V, int64_t D) {
  const int64_t i = blockIdx.x, v = ld_id(tok, i);
  const bool ok = v >= 0 && v < V;
  for (int64_t c = threadIdx.x; c < D; c += TOK_THREADS)
    from_f(out[i * D + c], ok ? to_f(w[v * w_stride + c]) * scale : __builtin_nanf(""));
}

template <typename T>
__global__ __launch_bounds__(TOK_THREADS) void k_embed_rows_bwd(Ids tok, const T* __restrict__ dout, int64_t d_stride,
                                                                float scale, int64_t padding, T* __restrict__ dw,
                                                                int64_t N, int64_t D) {
  const int64_t v = blockIdx.x, c = static_cast<int64_t>(blockIdx.y) * TOK_THREADS + threadIdx.x;
  float s = 0.f;
  if (v != padding)
    for (int64_t i = 0; i < N; ++i)
      if (ld_id(tok, i) == v && c < D) s += to_f(dout[i * d_stride + c]);
  if (c < D) from_f(dw[v * D + c], s * scale);
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
  GHM_CHECK(rows >= 0 && rows < (int64_t(1) << 31) && V >= 1 && V < (int64_t(1) << 31), "shape (rows, V < 2^31)"); \
  GHM_CHECK(n_inner >= 1 && s_outer >= 0 && s_inner >= 0, "row strides")

extern "C" int64_t ghm_token_logprobs_ws(int64_t rows, int64_t V, int top_k, int dtype) {
  (void)rows; (void)V; (void)top_k; (void)dtype;
  return 0;
}

extern "C" int ghm_token_logprobs(const void* logits, int dtype, int64_t n_inner, int64_t s_outer, int64_t s_inner,
                                  int64_t rows, int64_t V, const void* targets, int id_bits, int64_t ignore_index,
                                  int top_k, float* logprob, float* entropy, float* stats, float* top_logprob,
                                  int64_t* top_id, void* ws, int64_t ws_bytes, void* stream) {
  TOK_CHECK_ROWS();
  GHM_CHECK(top_k >= 0 && top_k <= GHM_TOP_MAX && top_k <= V, "top_k (0 .. min(64, V))");
  GHM_CHECK(!targets || ids_ok(id_bits), "id_bits (8, 32, 64)");
  GHM_CHECK(rows == 0 || (logits && (!targets || logprob) && (!logprob || targets) &&
                          (top_k == 0 || (top_logprob && top_id))), "null pointer");
  GHM_CHECK(ws_bytes >= ghm_token_logprobs_ws(rows, V, top_k, dtype), "workspace too small");
  (void)ws;
  if (rows == 0) return GHM_OK;
  const Rows m{logits, n_inner, s_outer, s_inner};
  const Ids t{targets, id_bits};
  TOK_DISPATCH(dtype, hipLaunchKernelGGL(k_score<T>, dim3(static_cast<unsigned>(rows)), dim3(TOK_THREADS), 0,
                                         ghm_stream(stream), m, static_cast<int>(V), t, ignore_index, top_k, logprob,
                                         entropy, reinterpret_cast<float2*>(stats), top_logprob, top_id));
  return ghm_launch_status();
}

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
  const Ids t{targets, id_bits};
  TOK_DISPATCH(dtype, hipLaunchKernelGGL(k_score_bwd<T>, dim3(static_cast<unsigned>(rows)), dim3(TOK_THREADS), 0,
                                         ghm_stream(stream), m, static_cast<int>(V), t, ignore_index,
                                         d_top ? top_k : 0, top_id, reinterpret_cast<const float2*>(stats), entropy,
                                         d_logprob, d_entropy, d_top, static_cast<T*>(dlogits)));
  return ghm_launch_status();
}

#define DISTILL_CHECK()                                                                                         \
  TOK_CHECK_ROWS();                                                                                             \
  GHM_CHECK(ids_ok(id_bits) && id_bits != 8 && dtype_ok(t_dtype), "top_ids (32 or 64 bits), top_logits dtype"); \
  GHM_CHECK(!targets || ids_ok(target_bits), "target_bits (8, 32, 64)");                                        \
  GHM_CHECK(k >= 1 && k <= GHM_DISTILL_MAX, "k (1 .. 1024)");                                                   \
  GHM_CHECK(temperature > 0.f && temperature <= FLT_MAX, "temperature");                                        \
  GHM_CHECK(alpha >= 0.f && alpha <= 1.f && (targets || alpha == 1.f), "alpha (0 .. 1; below 1 needs targets)")

extern "C" int64_t ghm_distill_ws(int64_t rows, int64_t V, int dtype) {
  (void)rows; (void)V; (void)dtype;
  return 0;
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
  GHM_CHECK(ws_bytes >= ghm_distill_ws(rows, V, dtype), "workspace too small");
  (void)ws;
  hipStream_t s = ghm_stream(stream);
  const Rows m{logits, n_inner, s_outer, s_inner};
  const Teacher tc{{top_ids, id_bits}, top_logits, t_dtype, k};
  const Ids t{targets, target_bits};
  float4* st = reinterpret_cast<float4*>(stats);
  const float* nm = reduction == 1 ? norm : nullptr;
  const dim3 g(static_cast<unsigned>(rows)), b(TOK_THREADS);
  if (nm) hipLaunchKernelGGL(k_distill_count, dim3(1), b, 0, s, tc, t, ignore_index, rows, norm);
  if (rows) {
    TOK_DISPATCH(dtype, hipLaunchKernelGGL(k_distill_rows<T>, g, b, 0, s, m, static_cast<int>(V), tc, t, ignore_index,
                                           temperature, alpha, row_loss, st));
    if (dlogits)
      TOK_DISPATCH(dtype, hipLaunchKernelGGL(k_distill_grad<T>, g, b, 0, s, m, static_cast<int>(V), tc, t,
                                             ignore_index, temperature, alpha, st, nm, nullptr, 0, grad_scale,
                                             static_cast<T*>(dlogits)));
  }
  if (reduction) hipLaunchKernelGGL(k_distill_total, dim3(1), b, 0, s, row_loss, rows, nm, loss);
  return ghm_launch_status();
}

extern "C" int ghm_distill_bwd(const void* logits, int dtype, int64_t n_inner, int64_t s_outer, int64_t s_inner,
                               int64_t rows, int64_t V, const void* top_ids, int id_bits, const void* top_logits,
                               int t_dtype, int k, const void* targets, int target_bits, int64_t ignore_index,
                               float temperature, float alpha, const float* stats, const float* norm,
                               const float* d_loss, int d_rows, void* dlogits, void* stream) {
  DISTILL_CHECK();
  GHM_CHECK(rows == 0 || (logits && top_ids && top_logits && stats && d_loss && dlogits), "null pointer");
  if (rows == 0) return GHM_OK;
  const Rows m{logits, n_inner, s_outer, s_inner};
  const Teacher tc{{top_ids, id_bits}, top_logits, t_dtype, k};
  const Ids t{targets, target_bits};
  TOK_DISPATCH(dtype, hipLaunchKernelGGL(k_distill_grad<T>, dim3(static_cast<unsigned>(rows)), dim3(TOK_THREADS), 0,
                                         ghm_stream(stream), m, static_cast<int>(V), tc, t, ignore_index, temperature,
                                         alpha, reinterpret_cast<const float4*>(stats), norm, d_loss, d_rows, 1.f,
                                         static_cast<T*>(dlogits)));
  return ghm_launch_status();
}

#define EMBED_CHECK()                                                                                              \
  GHM_CHECK(dtype_ok(dtype) && ids_ok(id_bits), "dtype (0 f32, 1 bf16, 2 f16), id_bits (8, 32, 64)");              \
  GHM_CHECK(N >= 0 && N < (int64_t(1) << 31) && V >= 1 && V < (int64_t(1) << 31) && D >= 1 && D < (int64_t(1) << 24), \
            "shape (N, V < 2^31, D < 2^24)")

extern "C" int ghm_embed_rows_fwd(const void* tokens, int id_bits, const void* weight, int dtype, int64_t w_stride,
                                  float scale, void* out, int64_t N, int64_t V, int64_t D, void* stream) {
  EMBED_CHECK();
  GHM_CHECK(w_stride >= 0, "row stride");
  GHM_CHECK(N == 0 || (tokens && weight && out), "null pointer");
  if (N == 0) return GHM_OK;
  TOK_DISPATCH(dtype, hipLaunchKernelGGL(k_embed_rows<T>, dim3(static_cast<unsigned>(N)), dim3(TOK_THREADS), 0,
                                         ghm_stream(stream), Ids{tokens, id_bits}, static_cast<const T*>(weight),
                                         w_stride, scale, static_cast<T*>(out), V, D));
  return ghm_launch_status();
}

extern "C" int64_t ghm_embed_rows_bwd_ws(int64_t N, int64_t V, int64_t D) {
  (void)N; (void)V; (void)D;
  return 0;
}

extern "C" int ghm_embed_rows_bwd(const void* tokens, int id_bits, const void* dout, int dtype, int64_t d_stride,
                                  float scale, int64_t padding_idx, void* dweight, int64_t N, int64_t V, int64_t D,
                                  void* ws, int64_t ws_bytes, void* stream) {
  EMBED_CHECK();
  GHM_CHECK(d_stride >= 0 && padding_idx >= -1 && padding_idx < V, "row stride, padding_idx (-1 .. V - 1)");
  GHM_CHECK(dweight && (N == 0 || (tokens && dout)), "null pointer");
  GHM_CHECK(ws_bytes >= ghm_embed_rows_bwd_ws(N, V, D), "workspace too small");
  (void)ws;
  TOK_DISPATCH(dtype, hipLaunchKernelGGL(k_embed_rows_bwd<T>,
                                         dim3(static_cast<unsigned>(V), static_cast<unsigned>((D + TOK_THREADS - 1) / TOK_THREADS)),
                                         dim3(TOK_THREADS), 0, ghm_stream(stream), Ids{tokens, id_bits},
                                         static_cast<const T*>(dout), d_stride, scale, padding_idx,
                                         static_cast<T*>(dweight), N, D));
  return ghm_launch_status();
}
