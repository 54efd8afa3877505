// The scaled embedding lookup and its gradient by sorted tokens.
#include "ghm_token.h"

namespace {

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

// A block takes `per` rows of `vecs` vectors; lanes take vectors in turn.  Bound by the
// writes: 16,384 tokens x 2048 bf16 in 17 us (67 MB each way, the read one mostly cached).
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void k_embed_rows(Ids tok, const T* __restrict__ weight, int64_t w_stride,
                                                    float scale, T* __restrict__ out, int64_t N, int64_t V, int D,
                                                    int vecs, int per) {
  constexpr int VE = Vec<T>::N, U = 4;
  const int64_t i0 = block_number() * per;
  if (i0 >= N) return;
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

// The same for large outputs whose rows are not whole lines (D >= VE): the output is one run of
// N * D values in vectors of VE from its first 16-byte boundary on, 256 * U of them per
// block, so that lines are written whole and past the caches, whatever D is.  A vector that crosses
// from a row into the next is put together from the one's last VE values and the other's
// first.  131,071 x 1001 f32 in 102 us (5.1 TB/s; 129 row by row; 144 us right after a gradient
// of the same size, whose lines are still to be written back), 131,071 x 2047 bf16
// in 114 (151); what fits the 256 MB cache is sooner there by rows: 10,000 x 1001 f32 in 11 us
// (21), 100,000 x 1001 bf16 in 41 (51).
constexpr int64_t RUN_BYTES = int64_t(1) << 28;
template <typename T>
__global__ __launch_bounds__(256) void k_embed_run(Ids tok, const T* __restrict__ weight, int64_t w_stride, float scale,
                                                   T* __restrict__ out, int64_t N, int64_t V, uint32_t D, int head,
                                                   int64_t vecs) {
  constexpr int VE = Vec<T>::N, U = 4;
  using raw = typename Vec<T>::raw;
  const auto start = [&](int64_t t) { return weight + (t >= 0 && t < V ? t : 0) * w_stride; };  // a bad token reads row 0
  const auto factor = [&](int64_t t) { return t >= 0 && t < V ? scale : __builtin_nanf(""); };
  const int64_t j0 = block_number() * (256 * U), e0 = head + j0 * VE, r0 = e0 / D;
  if (j0 >= vecs) return;
  if (j0 == 0) {  // the values before the first vector and after the last one
    const int t = threadIdx.x;
    const int64_t e = t < head ? t : head + vecs * VE + t - head;
    if (t < head + VE && e < N * D) {
      const int64_t v = ld_id(tok, e / D);
      from_f(out[e], to_f(start(v)[e % D]) * factor(v));
    }
  }
  const uint32_t c0 = static_cast<uint32_t>(e0 - r0 * D);
  int64_t v[U], next[U];
  uint32_t col[U], row[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {  // past the end: the last vector again
    const int64_t j = j0 + threadIdx.x + 256 * u;
    const uint32_t o = c0 + static_cast<uint32_t>((j < vecs ? j : vecs - 1) - j0) * VE;
    row[u] = o / D;
    col[u] = o - row[u] * D;
  }
  ld_ids<U>(tok, v, [&](int u) { return r0 + row[u]; });
  ld_ids<U>(tok, next, [&](int u) { return r0 + row[u] + 1 < N ? r0 + row[u] + 1 : N - 1; });
  u32x4 x[U], y[U];
  bool in[U];
  const auto scaled = [&](u32x4 p, float f) {
    float z[VE];
    T e[VE];
    unpack<T>(p, z);
#pragma unroll
    for (int i = 0; i < VE; ++i) from_f(e[i], z[i] * f);
    __builtin_memcpy(&p, e, 16);
    return p;
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    in[u] = col[u] + VE <= D;
    x[u] = *reinterpret_cast<const raw*>(start(v[u]) + (in[u] ? col[u] : D - VE));
  }
#pragma unroll
  for (int u = 0; u < U; ++u) y[u] = in[u] ? x[u] : *reinterpret_cast<const raw*>(start(next[u]));
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t j = j0 + threadIdx.x + 256 * u;
    if (j >= vecs) break;
    u32x4 o = scaled(x[u], factor(v[u]));
    if (!in[u]) {
      const u32x4 q = scaled(y[u], factor(next[u]));
      const uint32_t k = col[u] - (D - VE), words = k * sizeof(T) / 4;  // k values of x[u] are before this vector
      uint32_t z[8] = {o[0], o[1], o[2], o[3], q[0], q[1], q[2], q[3]};
#pragma unroll
      for (int i = 0; i < 6; ++i) z[i] = words & 2 ? z[i + 2] : z[i];
#pragma unroll
      for (int i = 0; i < 5; ++i) z[i] = words & 1 ? z[i + 1] : z[i];
      if (sizeof(T) == 2 && (k & 1)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = z[i] >> 16 | z[i + 1] << 16;
      }
      o = u32x4{z[0], z[1], z[2], z[3]};
    }
    __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(out + head + j * VE));
  }
}

// ---------------------------------------------------------------------------
// Its gradient dW_v = scale sum_{i: tok_i = v} dout_i.  The positions are sorted by token
// (stable radix sort, so a token's positions stay in order); chunks of the sorted list are
// summed in f32, a token that crosses chunks through partial rows joined in order; table
// rows without a token are written 0 beside it.  No atomics on values: a fixed order.
// ---------------------------------------------------------------------------
constexpr int SORT_BITS = 9, SORT_BINS = 1 << SORT_BITS, SORT_ROUNDS = 4;
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
// Bound by the reads and writes: 16,384 x 2048 bf16 into 65,536 rows in 60 us (335 MB, 5.6
// TB/s), 131,071 x 1001 f32 in about 120 us (545 MB, 4.5 TB/s); the sorts before them take
// 25 and 35 us, the joins 6 and 7.
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
  // Rows are read one step ahead of their sums and kept packed; their keys and positions are read
  // in the same step, so that each step's row loads wait for its position loads (16 bytes each:
  // chunks are multiples of U, and the arrays are padded).  Entries past the end take row 0 and
  // are not used.
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

// Tables of at most FEW_V rows (the model's own 10 token values) need no sort: a block keeps
// the sums of its positions for all rows in LDS, each column one lane's, in order; the
// blocks' sums are joined in order by a second launch, which writes every row.  10,368
// positions of 10 x 256 f32: 17 us, by the sort (three launches) 31; 32,768 x 1024: 43 and
// 53; where there is more to read, the LDS sums of one row at a time fall behind (131,071 x
// 1024 bf16 into 32 rows: 160 and 81), so up to FEW_ELEMS values only.
constexpr int FEW_V = 32, FEW_BLOCKS = 256, FEW_JOIN = 16, FEW_ELEMS = 1 << 24;
inline bool few_rows(int64_t N, int64_t V, int64_t D) { return V <= FEW_V && N * D <= FEW_ELEMS; }
template <typename T>
__global__ __launch_bounds__(256) void k_embed_few(Ids tok, const T* __restrict__ dout, int64_t d_stride, int64_t pad,
                                                   int V, int64_t N, int D, int64_t per, float* __restrict__ parts) {
  constexpr int C = 4 / sizeof(T), U = 8;  // columns per lane: 4 bytes of a row
  extern __shared__ float sum[];  // [V][256 C]
  const int64_t lo = blockIdx.x * per, hi = lo + per < N ? lo + per : N;
  const int col0 = (blockIdx.y * 256 + threadIdx.x) * C;
  const int col = col0 + C <= D || D < C ? col0 : D - C;  // an odd last column is shared with the one before
  if (col0 >= D) return;
  float* mine = sum + threadIdx.x * C;
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int c = 0; c < C; ++c) mine[v * 256 * C + c] = 0.f;
  for (int64_t i = lo; i < hi; i += U) {
    int64_t v[U];
    T x[U][C];
    const auto at = [&](int u) { return i + u < hi ? i + u : hi - 1; };
    ld_ids<U>(tok, v, at);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const T* row = dout + at(u) * d_stride + col;
#pragma unroll
      for (int c = 0; c < C; ++c) x[u][c] = row[col + c < D ? c : 0];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= hi || v[u] < 0 || v[u] >= V || v[u] == pad) continue;
#pragma unroll
      for (int c = 0; c < C; ++c) mine[v[u] * 256 * C + c] += to_f(x[u][c]);
    }
  }
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (col + c < D) parts[(static_cast<int64_t>(blockIdx.x) * V + v) * D + col + c] = mine[v * 256 * C + c];
}
// row v = blockIdx.x, 64 columns per block: FEW_JOIN waves take the blocks' sums in turn
template <typename T>
__global__ __launch_bounds__(64 * FEW_JOIN) void k_embed_few_join(const float* __restrict__ parts, int blocks, int V, int D,
                                                                  float scale, T* __restrict__ dw) {
  __shared__ float red[FEW_JOIN][64];
  const int v = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6, col = blockIdx.y * 64 + lane;
  const int per = (blocks + FEW_JOIN - 1) / FEW_JOIN, a = w * per, b = a + per < blocks ? a + per : blocks;
  float s = 0.f;
  if (col < D) {
#pragma unroll 16
    for (int j = a; j < b; ++j) s += parts[(static_cast<int64_t>(j) * V + v) * D + col];
  }
  red[w][lane] = s;
  __syncthreads();
  if (w != 0 || col >= D) return;
#pragma unroll
  for (int j = 1; j < FEW_JOIN; ++j) s += red[j][lane];
  from_f(dw[static_cast<int64_t>(v) * D + col], s * scale);
}

// no token at all: every table row is 0
template <typename T>
__global__ __launch_bounds__(256) void k_embed_zero(T* __restrict__ dw, int64_t n) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
    from_f(dw[i], 0.f);
}

}  // namespace

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
  const dim3 g = grid_of((N + per - 1) / per, 256), b(256);
  const Ids t{tokens, id_bits};
  const int d = static_cast<int>(D);
  hipStream_t s = ghm_stream(stream);
  const int64_t size = 16 / ve;
  if (!whole_lines(out, D * size) && D >= ve && N * D * size > RUN_BYTES) {
    const int head = static_cast<int>((16 - reinterpret_cast<uintptr_t>(out) % 16) % 16 / size);
    const int64_t run = (N * D - head) / ve;
    TOK_DISPATCH(dtype, hipLaunchKernelGGL(k_embed_run<T>, grid_of((run + 1023) / 1024, 256), b, 0, s, t,
                                           static_cast<const T*>(weight), w_stride, scale, static_cast<T*>(out), N, V,
                                           static_cast<uint32_t>(D), head, run));
  } else if (whole_lines(out, D * size))
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
  p.counts = at, at += up256((N / (64 * 8 * SORT_ROUNDS) + 2) * SORT_BINS * 4);
  p.used = at, at += up256(p.used_words * 4);
  p.parts = at, at += up256(p.chunks * 2 * D * 4);
  p.bytes = at;
  return p;
}

// blocks of k_embed_few: 32 positions each at least; the last one is not empty
inline int few_blocks(int64_t N) {
  const int64_t b = (N + 31) / 32 < FEW_BLOCKS ? (N + 31) / 32 : FEW_BLOCKS, per = (N + b - 1) / b;
  return static_cast<int>((N + per - 1) / per);
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
  if (few_rows(N, V, D)) {
    const int blocks = few_blocks(N);
    const int64_t per = (N + blocks - 1) / blocks;
    float* sums = reinterpret_cast<float*>(ws);
    constexpr int cols = 256 * (4 / sizeof(T));
    hipLaunchKernelGGL(k_embed_few<T>, dim3(blocks, static_cast<unsigned>((D + cols - 1) / cols)), dim3(256),
                       static_cast<unsigned>(V * cols * 4), s, tok,
                       dout, d_stride, pad, static_cast<int>(V), N, D, per, sums);
    hipLaunchKernelGGL(k_embed_few_join<T>, dim3(static_cast<unsigned>(V), static_cast<unsigned>((D + 63) / 64)),
                       dim3(64 * FEW_JOIN), 0, s, sums, blocks, static_cast<int>(V), D, scale, dw);
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
  } else if (N <= 64 * 8 * SORT_ROUNDS * SORT_TILES) {
    launch_sort<8, SORT_SUM>(p, tok, pad, N, V, ws, s);
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
  if (few_rows(N, V, D)) return up256(static_cast<int64_t>(few_blocks(N)) * V * D * 4);
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
