// Distillation from a teacher's top logits, mixed with hard labels: row losses, their
// reduction, and the gradient -- in the same launch as the loss, or from saved statistics.
#include "ghm_token.h"

namespace {

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
// 8 entries of a row for one lane, none waiting for another (one by one, 10,240 rows of 10
// values and 4 entries took 10.5 us in place of 7.8)
struct Entries {
  int64_t id[8];
  float t[8];
  bool has[8];
};
__device__ __forceinline__ Entries ld_entries(const Teacher& tc, int64_t first, int j0) {
  Entries e;
  const auto at = [&](int u) { return first + (j0 + u < tc.k ? j0 + u : tc.k - 1); };
  ld_ids<8>(tc.ids, e.id, at);
  if (tc.dtype == 0) {
#pragma unroll
    for (int u = 0; u < 8; ++u) e.t[u] = static_cast<const float*>(tc.logits)[at(u)];
  } else if (tc.dtype == 1) {
#pragma unroll
    for (int u = 0; u < 8; ++u) e.t[u] = to_f(static_cast<const bf16_t*>(tc.logits)[at(u)]);
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u) e.t[u] = to_f(static_cast<const f16_t*>(tc.logits)[at(u)]);
  }
#pragma unroll
  for (int u = 0; u < 8; ++u) e.has[u] = j0 + u < tc.k && e.id[u] >= 0 && !(e.t[u] == NEG_INF);
  return e;
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
      for (int j0 = 0; j0 < t.k && !in; j0 += 8) {
        const Entries e = ld_entries(t, r * t.k, j0);
#pragma unroll
        for (int u = 0; u < 8; ++u) in |= e.has[u];
      }
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

// A row that is NaN, loss and gradient: an entry or the target lies outside the vocabulary, or the row
// has no distribution (no finite maximum: the logarithm of its sum, l2, is not finite).
__device__ __forceinline__ bool row_bad(bool bad_entry, const Ids& targets, int64_t y, int V, float l2) {
  return bad_entry || (targets.p && (y < 0 || y >= V)) || !(l2 - l2 == 0.f);
}
// the factor of the teacher's part of the gradient: none without entries, but a row that is NaN stays so
__device__ __forceinline__ float teacher_scale(const Mix& mix, bool some, float scale) {
  if (scale != scale) return scale;
  return some && mix.alpha != 0.f ? scale * mix.alpha * mix.tau : 0.f;
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
  g.A = teacher_scale(mix, some, scale);
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
    if (g.A != 0.f) v -= g.A * q;  // without the teacher's part its logits are not used, NaN or not
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
  if (g.two) map_row<T, N, U, W, true, false>(z, d, lo, hi, w, lane, [=](float x) { return g.both(x); });
  else map_row<T, N, U, W, true, false>(z, d, lo, hi, w, lane, [=](float x) { return g.one(x); });
  group_sync<W>();
  distill_entries<T, W>(z, d, lo, hi, tc, mix, g, lds, y, w, lane);
}

// Sums of a row, its loss, and its gradient if dz is there, by a group of W waves.  The
// gradient reads the row again; its stores go past the caches so that the row is still in
// the 256 MB one: 4,096 rows of 131,072 bf16 values, 64 entries, in 495 us (4.3 TB/s of one
// read and one write; 553 us with ordinary stores).  That needs few enough rows in flight:
// 16 waves on a row of more than 8,192 vectors (8 waves: 524 us), 8 on shorter ones.
// Without a gradient 189 us (5.7 TB/s).
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
  const int64_t r = block_number() * G + wave / W;
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
  const bool bad = row_bad(tr.bad, targets, y, V, l2);
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
// lane, R * 64 * W * N values at most): the logits are read once.  For rows of up to 4,096
// vectors: 4,194 rows of 16,000 bf16 values with two softmaxes 68 us (3.9 TB/s, the two
// exponentials twice per value), read twice 82; on longer ones a CU holds too few rows to
// load one while it computes another (131,072 values: 590 us against 495).
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
  const int64_t r = block_number() * G + wave / W;
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
  const bool bad = row_bad(tr.bad, targets, y, V, l2);
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
    row_loss[r] = row_bad(tr.bad, targets, y, V, l2) ? __builtin_nanf("") : loss;
    row_stats[r] = make_float4(a.m, l1, l2, 1.f);
  }
}
// ... and the gradient from the row's statistics, the last rows first (what the sums read last is
// still in the 256 MB cache: loss and gradient of 2,048 rows of 65,536 f32 values 297 us, 316 in order)
template <typename T, int N, int U, int W>
__global__ __launch_bounds__(256) void k_distill_grad(Rows rows, int64_t n_rows, int V, Teacher tc, Ids targets,
                                                      int64_t ignore, Mix mix, Upstream up, int parts, int part_len,
                                                      const float4* __restrict__ row_stats, T* __restrict__ dz) {
  constexpr int G = 4 / W;
  __shared__ float teach_slots[G][4 * W];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, w = wave % W;
  const int64_t item = n_rows * parts - 1 - (block_number() * G + wave / W);
  if (item < 0) return;
  const int64_t r = item / parts;
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
  const bool bad = row_bad(tr.bad, targets, y, V, st.z);
  distill_row_grad<T, N, U, W>(
      row_ptr<T>(rows, r), d, lo, hi, tc, mix,
      distill_grad(mix, tr.some, st.x, st.y, st.z, bad ? __builtin_nanf("") : upstream(up, r, lane)), lds, y, w, lane);
}

// Rows of at most SHORT_V values, one lane per row: loss, statistics and gradient, each
// if asked for.
template <typename T, int M>
__global__ __launch_bounds__(64) void k_distill_short(Rows rows, int64_t n_rows, int V, Teacher tc, Ids targets,
                                                      int64_t ignore, Mix mix, Upstream up,
                                                      float* __restrict__ row_loss, float4* __restrict__ row_stats,
                                                      T* __restrict__ dz) {
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * 64 + threadIdx.x;
  const bool live = r0 < n_rows;
  const int64_t r = live ? r0 : n_rows - 1, first = r * tc.k;
  float scale = dz ? upstream(up, r, threadIdx.x) : 0.f;  // by the whole wave
  if (!live) return;
  const int64_t y = targets.p ? ld_id(targets, r) : -1;
  float x[M];
  {
    const T* z = row_ptr<T>(rows, r);  // padding rows are read and not used
#pragma unroll
    for (int v = 0; v < M; ++v) x[v] = v < V ? to_f(z[v]) : NEG_INF;
  }
  float mt = -FLT_MAX;
  bool some = false, bad = false;
  for (int j0 = 0; j0 < tc.k; j0 += 8) {
    const Entries e = ld_entries(tc, first, j0);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      some |= e.has[u];
      bad |= e.has[u] && e.id[u] >= V;
      mt = e.has[u] ? fmaxf(mt, e.t[u]) : mt;
    }
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
  float q[M];
  Sums a;
#pragma unroll
  for (int v = 0; v < M; ++v) {
    a.m = fmaxf(a.m, x[v]);
    q[v] = 0.f;
  }
  fold<SECOND_EXP, true>(a, x, LOG2E, mix.c2);
  const float l1 = a.log_s(), l2 = a.log_t();
  bad = row_bad(bad, targets, y, V, l2);
  float st = 0.f, kl = 0.f;
  for (int j0 = 0; j0 < tc.k; j0 += 8) {
    const Entries e = ld_entries(tc, first, j0);
#pragma unroll
    for (int u = 0; u < 8; ++u) st += e.has[u] ? __builtin_amdgcn_exp2f((e.t[u] - mt) * mix.it * LOG2E) : 0.f;
  }
  const float lt = logf(st);
  for (int j0 = 0; j0 < tc.k; j0 += 8) {
    const Entries e = ld_entries(tc, first, j0);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (!e.has[u]) continue;
      const float lq = (e.t[u] - mt) * mix.it - lt, qj = __builtin_amdgcn_exp2f(lq * LOG2E);
      float zi = 0.f;
#pragma unroll
      for (int v = 0; v < M; ++v) {
        q[v] += v == e.id[u] ? qj : 0.f;
        zi = v == e.id[u] ? x[v] : zi;
      }
      if (!(qj == 0.f)) kl += qj * (lq - ((zi - a.m) * mix.it - l2));
    }
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
  const float A = teacher_scale(mix, some, scale);
  const float B = mix.hard ? scale * (1.f - mix.alpha) : 0.f;
#pragma unroll
  for (int v = 0; v < M; ++v) {
    if (v >= V) break;
    const float d = x[v] - a.m;
    float g = A == 0.f ? 0.f : A * (__builtin_amdgcn_exp2f(__builtin_fmaf(d, mix.c2, -l2 * LOG2E)) - q[v]);
    if (mix.hard) g += B * (__builtin_amdgcn_exp2f(__builtin_fmaf(d, LOG2E, -l1 * LOG2E)) - (v == y ? 1.f : 0.f));
    from_f(dz[r * V + v], g);
  }
}

}  // namespace

#define DISTILL_CHECK()                                                                                         \
  TOK_CHECK_ROWS();                                                                                             \
  GHM_CHECK(ids_ok(id_bits) && id_bits != 8 && dtype_ok(t_dtype), "top_ids (32 or 64 bits), top_logits dtype"); \
  GHM_CHECK(!targets || ids_ok(target_bits), "target_bits (8, 32, 64)");                                        \
  GHM_CHECK(k >= 1 && k <= GHM_DISTILL_MAX, "k (1 .. 1024)");                                                   \
  GHM_CHECK(temperature >= 1e-6f && temperature <= 1e6f, "temperature (1e-6 .. 1e6)");                 \
  GHM_CHECK(alpha >= 0.f && alpha <= 1.f && (targets || alpha == 1.f || rows == 0), "alpha (0 .. 1; below 1 needs targets)")

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
  const dim3 g = grid_of((a.rows + G - 1) / G, 64 * G * W), b(64 * G * W);
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
  const dim3 g = grid_of((a.rows + G - 1) / G, 64 * G * W), b(64 * G * W);
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
  hipLaunchKernelGGL((k_distill_grad<T, N, U, W>), grid_of((a.rows * p.parts + G - 1) / G, 256), dim3(256), 8 * a.tc.k * G,
                     a.s, a.m, a.rows, a.V, a.tc, a.t, a.ignore, a.mix, up, p.parts, p.len, a.stats, dz);
}
template <typename T>
void distill_short(const Distill& a, const Upstream& up, float* row_loss, T* dz) {
  const dim3 g(static_cast<unsigned>((a.rows + 63) / 64)), b(64);
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
  const Split p = row_split(a.rows, a.V, N, dz ? SPLIT_STEP : SPLIT_SUMS);
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
    else if (nv <= 512 && a.rows >= 1024) launch_step<T, 8, 1>(a, up, dz);
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
  if (rows <= 0 || V <= 0) return DISTILL_WS_HEAD;
  const Split p = row_split(rows, V, dtype == 0 ? 4 : 8, {SPLIT_STEP.vectors, SPLIT_SUMS.rows});  // either rule's
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
