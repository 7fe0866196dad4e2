// Beam search on the GPU: the best candidates over beams and vocabulary, and beams that go on from another beam's keys, values and
// states.
//
// CodeClaper/tinyllama.c samples one sequence's next token on the host (sampler.c:107-257) and has no search over several.
// A candidate is a pair of beam k and token v of a request, of value
//     c_kv = s_k + x_kv - log(sum_u exp x_ku),
// and the n best of a request's K * V are wanted, equal values by the lowest k * V + v.  Two kernels:
//   * beam_scan_kernel reads every logit once.  A warp takes a piece of a row, 64 (or 16) values a lane in registers, and leaves the
//     piece's maximum and its sum of exponentials; nothing crosses warps.
//   * beam_merge_kernel, a block a request, makes the rows' logarithms of sums.  The n-th largest of the pieces' maxima bounds the n best from below,
//     so that only the pieces whose maximum reaches it (n to 2 n of hundreds, by a threshold that a few counts find) can hold
//     any: those are read again, a warp each, and what reaches the threshold is ranked by counting.  (With the n largest of every piece
//     left by the first kernel it took twice as long: 34 of 66 us went into values that no request wanted.)
// Bound by HBM for a batch (192 rows of 130,048 logits: 100 MB in 16.5 us, 6.1 TB/s; the merge, 16 candidates of 32 requests, some 9 more, of which
// half are trips to the L2 and half the counts that find the threshold), by the two launches for one request (7.4 us for 4 rows of 65,536).
// Arithmetic: exponentials and sums in 32 bits over 16 values at most, the sums of those, the logarithm and the values that are compared in
// 64 bits: two candidates change places only where they are nearer than the 2^-22 or so that this leaves.
#include "common.cuh"
#include <type_traits>

namespace {

constexpr int MAX_N = 64;                // candidates of a request
constexpr int MAX_BEAMS = 64;
constexpr int SCAN_WARPS = 4;
constexpr int MERGE_T = 512, MERGE_WARPS = MERGE_T / 32;
constexpr int MERGE_CAP = 4096;          // values that may reach the threshold; more equal ones are taken one after the other
constexpr int MERGE_RANK = 512;          // and of which so many are ranked side by side, after a second threshold
constexpr int MERGE_LISTS = 512;         // pieces that reach the threshold and are shared out evenly
constexpr int SHARES = 16;               // parts of a request's logits where values are taken one after the other
constexpr int MAX_LISTS = 36864;         // pieces of a request: a word of shared memory each

struct Stats { double sum; float max; int pad; };      // of a piece: sum exp(x - max) and max

// larger float <=> larger unsigned
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ bool alive(const float* scores, const unsigned char* ended, int row) {
  return isfinite(scores[row]) && !(ended && ended[row]);
}

// A piece's values, VPL a lane: index_of(q) = (q / VEC * 32 + lane) * VEC + q % VEC; -infinity behind the row's end (left: values from
// the piece's start on).  VEC 4: the row starts on a 16-byte boundary.
template <int VPL, int VEC>
__device__ __forceinline__ void load_piece(const float* __restrict__ x, int left, int lane, float (&v)[VPL]) {
  if (left >= 32 * VPL) {
#pragma unroll
    for (int q = 0; q < VPL; q += VEC) {
      if constexpr (VEC == 4) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(x) + q / 4 * 32 + lane);
        v[q] = f.x; v[q + 1] = f.y; v[q + 2] = f.z; v[q + 3] = f.w;
      } else v[q] = __ldcs(x + q * 32 + lane);
    }
  } else {
#pragma unroll
    for (int q = 0; q < VPL; q++) {
      const int at = (q / VEC * 32 + lane) * VEC + q % VEC;
      v[q] = at < left ? __ldcs(x + at) : -INFINITY;
    }
  }
}

// grid: pieces of all rows, SCAN_WARPS a block.
template <int VPL, int VEC>
__global__ void __launch_bounds__(SCAN_WARPS * 32)
beam_scan_kernel(const float* __restrict__ logits, long long ld, const float* __restrict__ scores, const unsigned char* __restrict__ ended,
                 int rows, int V, int n_pieces, Stats* __restrict__ stats) {
  asm volatile("griddepcontrol.launch_dependents;");
  tlc_wait(logits, scores, ended, stats);
  const int lane = threadIdx.x & 31;
  const long long piece = (long long)blockIdx.x * SCAN_WARPS + (threadIdx.x >> 5);
  const int row = (int)(piece / n_pieces), base = (int)(piece % n_pieces) * 32 * VPL;
  if (row >= rows || !alive(scores, ended, row)) return;
  float v[VPL];
  load_piece<VPL, VEC>(logits + (size_t)row * ld + base, V - base, lane, v);
  float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};          // (a NaN is nobody's maximum; it shows in the sum)
#pragma unroll
  for (int q = 0; q < VPL; q++) part[q % 4] = fmaxf(part[q % 4], v[q]);
  const float m = warp_max(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]))), top = m == -INFINITY ? 0.f : m;
  // (the largest is taken off first: a multiple of it would bring its own rounding into every term)
  double sum = 0.0;
#pragma unroll
  for (int g = 0; g < VPL; g += 16) {
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int q = g; q < g + 16; q += 2) {
      a += ex2((v[q] - top) * 1.4426950408889634f);
      b += ex2((v[q + 1] - top) * 1.4426950408889634f);
    }
    sum += (double)(a + b);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) stats[piece] = Stats{sum, m, 0};
}

// Candidates by value, equal ones by index.
__device__ __forceinline__ bool better(double a, int ai, double b, int bi) { return a > b || (a == b && ai < bi); }

template <int VPL, int VEC>
__global__ void __launch_bounds__(MERGE_T)
beam_merge_kernel(const float* __restrict__ logits, long long ld, const float* __restrict__ scores, const unsigned char* __restrict__ ended, int K,
                  int V, int n_pieces, int n, int pad, int placed, const Stats* __restrict__ stats, int* __restrict__ tokens,
                  int* __restrict__ parents, float* __restrict__ out_scores) {
  tlc_pdl(logits, scores, ended, stats, tokens, parents, out_scores);
  extern __shared__ int merge_room[];
  float* const c_value = reinterpret_cast<float*>(merge_room);           // [MERGE_CAP] logits that reach the threshold
  int* const c_index = merge_room + MERGE_CAP;                           // [MERGE_CAP] k * V + v of them; of ended beams -1 - k
  unsigned* const heads = reinterpret_cast<unsigned*>(merge_room + 2 * MERGE_CAP);     // of every piece: what its maximum is worth, as an ordered integer
  __shared__ double s_off[MAX_BEAMS], s_top[MAX_BEAMS], s_value[MERGE_RANK], s_best[MERGE_WARPS];
  __shared__ int s_index[MERGE_RANK], s_at[MERGE_WARPS], s_count, s_ranked, s_alive[MAX_BEAMS], s_list[MERGE_LISTS], s_lists, s_reach[2];
  __shared__ unsigned s_least;
  __shared__ double s_out[MAX_N], s_share[SHARES];
  __shared__ int s_out_at[MAX_N], s_share_at[SHARES];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, lists = K * n_pieces;
  if (tid == 0) s_count = s_lists = s_ranked = s_reach[0] = s_reach[1] = 0;
  // a logit x of row k is worth s_off + (x - s_top), with the row's largest in s_top and the beam's score less the logarithm of the sum of
  // exp(x - s_top) in s_off (one number for both would lose the score where a row holds nothing but the lowest number)
  for (int k = warp; k < K; k += MERGE_WARPS) {
    const int row = r * K + k;
    const Stats* st = stats + (size_t)row * n_pieces;
    float m = -INFINITY;
    for (int i = lane; i < n_pieces; i += 32) m = fmaxf(m, st[i].max);   // (of a row that is not alive whatever is there)
    bool on = alive(scores, ended, row);
    double off = 0.0;
    if (on) {
      m = warp_max(m);
      double sum = 0.0;
      for (int i = lane; i < n_pieces; i += 32) {
        const Stats a = st[i];
        // (a piece of nothing but -infinity and NaN: its sum is 0 or NaN)
        sum += a.max == -INFINITY ? (a.sum != a.sum ? a.sum : 0.0) : a.sum * exp((double)a.max - (double)m);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      off = (double)scores[row] - log(sum);
      on = isfinite(off);                              // no candidates of a row with a NaN, an infinity or nothing in it
    }
    if (lane == 0) { s_off[k] = off; s_top[k] = m; s_alive[k] = on; }
  }
  __syncthreads();
  auto worth_of = [&](int k, float x) { return s_off[k] + ((double)x - s_top[k]); };
  auto key_of = [&](int k, float x) { return ordered((float)worth_of(k, x)); };
  const Stats* const mine = stats + (size_t)r * lists;
  for (int l = tid; l < lists; l += MERGE_T) {
    const int k = l / n_pieces;
    unsigned h = 0;
    if (s_alive[k]) {
      const float m = mine[l].max;
      if (m > -INFINITY) h = key_of(k, m);
    }
    heads[l] = h;
  }
  __syncthreads();
  // a threshold that at least n of the pieces' maxima reach (and 2 n at most, where that can be found)
  if (warp == 0) {
    constexpr int HELD = 16;                           // of the first 512 pieces in registers
    unsigned held[HELD], least = 0xffffffffu, above = 0;
#pragma unroll
    for (int i = 0; i < HELD; i++) {
      held[i] = i * 32 + lane < lists ? heads[i * 32 + lane] : 0u;
      if (i * 32 + lane < lists) least = min(least, held[i]);
      above = max(above, held[i]);
    }
    for (int l = HELD * 32 + lane; l < lists; l += 32) { least = min(least, heads[l]); above = max(above, heads[l]); }
    least = __reduce_min_sync(0xffffffffu, least);
    above = __reduce_max_sync(0xffffffffu, above);
    if (lists < n) least = 0;
    else
      while (least < above) {                          // (least is reached by n, above + 1 by none)
        const unsigned trial = least + (above - least + 1) / 2;       // (at least 1: what is past the lists does not count)
        int reach = 0;
#pragma unroll
        for (int i = 0; i < HELD; i++) reach += held[i] >= trial;
        for (int l = HELD * 32 + lane; l < lists; l += 32) reach += heads[l] >= trial;
        reach = __reduce_add_sync(0xffffffffu, reach);
        if (reach >= n) least = trial; else above = trial - 1;
        if (reach >= n && reach <= 2 * n) break;
      }
    if (lane == 0) s_least = max(least, 1u);
  }
  __syncthreads();
  unsigned least = s_least;
  // a threshold of `low` or more that at least n and, where that can be found, at most `enough` of the block's keys reach
  auto search = [&](const auto& keys, unsigned low, int enough) {
    unsigned high = 0xffffffffu;
    __syncthreads();
    if (tid == 0) s_reach[0] = s_reach[1] = 0;
    __syncthreads();
    for (int turn = 0; low < high; turn++) {
      const unsigned trial = low + (high - low) / 2 + 1;
      int reach = 0;
#pragma unroll
      for (int i = 0; i < (int)(sizeof(keys) / sizeof(keys[0])); i++) reach += keys[i] >= trial;
      reach = __reduce_add_sync(0xffffffffu, reach);
      if (lane == 0) atomicAdd(&s_reach[turn & 1], reach);
      __syncthreads();
      reach = s_reach[turn & 1];
      if (tid == 0) s_reach[(turn + 1) & 1] = 0;
      __syncthreads();
      if (reach >= n) low = trial; else high = trial - 1;
      if (reach >= n && reach <= enough) break;
    }
    return low;
  };
  // the pieces that reach it, again
  for (int l = tid; l < lists; l += MERGE_T)
    if (heads[l] >= least) {
      const int at = atomicAdd(&s_lists, 1);
      if (at < MERGE_LISTS) s_list[at] = l;
    }
  __syncthreads();
  const int passing = s_lists;
  auto push = [&](double value, float logit, int index, int mark) {
    const int at = atomicAdd(&s_count, 1);             // (in any order: they are ranked below)
    if (at < MERGE_CAP) { c_value[at] = logit; c_index[at] = mark; }
    if (at < MERGE_RANK) { s_value[at] = value; s_index[at] = index; }
  };
  auto collect = [&](int l) {
    const int k = l / n_pieces, base = l % n_pieces * 32 * VPL;
    const float* const x = logits + (size_t)(r * K + k) * ld + base;
    float v[VPL];
    load_piece<VPL, VEC>(x, V - base, lane, v);
    // (the threshold as a logit of row k, a little lower: whatever is worth as much passes, and what is worth hardly less does no harm)
    const float worth = __uint_as_float(least & 0x80000000u ? least & 0x7fffffffu : ~least);
    // (never below the lowest number: load_piece has -infinity behind a row's end, and a threshold under every number's key is worth a NaN)
    constexpr float LOWEST = -3.402823466e38f;
    const float exact = (float)((double)worth - s_off[k] + s_top[k]), bar = least == 1u ? LOWEST : fmaxf(LOWEST, exact - 1e-6f * (fabsf(exact) + fabsf(worth)));
    // which of them reach it; those few are read once more (a body for each of 64 values would not fit the instruction cache)
    unsigned long long who = 0;
#pragma unroll
    for (int q = 0; q < VPL; q++) who |= (unsigned long long)(v[q] >= bar) << q;
    for (; who != 0; who &= who - 1) {
      const int q = __ffsll((long long)who) - 1, at = (q / VEC * 32 + lane) * VEC + q % VEC;
      const float f = x[at];
      push(worth_of(k, f), f, k * V + base + at, k * V + base + at);
    }
  };
  // Fewer pieces than n hold anything (one beam is alive: 15 pieces of 30,000 logits for 16 candidates), or those that reach the threshold
  // hold more than there is room for: then the maxima of the pieces' lanes make the threshold (64 such requests: 830 us one value after the
  // other, 18 this way).
  const bool few = passing * 32 <= MERGE_CAP;
  bool finer = few && least == 1u && passing * 32 * VPL > MERGE_CAP;
  int count;
  for (;;) {
    if (finer) {
      unsigned* const tops = reinterpret_cast<unsigned*>(c_value);       // [32 * passing]
      for (int i = warp; i < passing; i += MERGE_WARPS) {
        const int l = s_list[i], k = l / n_pieces, base = l % n_pieces * 32 * VPL;
        float v[VPL], m = -INFINITY;
        load_piece<VPL, VEC>(logits + (size_t)(r * K + k) * ld + base, V - base, lane, v);
#pragma unroll
        for (int q = 0; q < VPL; q++) m = fmaxf(m, v[q]);
        tops[i * 32 + lane] = m > -INFINITY ? key_of(k, m) : 0u;
      }
      __syncthreads();
      unsigned held[MERGE_CAP / MERGE_T];
#pragma unroll
      for (int i = 0; i < MERGE_CAP / MERGE_T; i++) held[i] = i * MERGE_T + tid < passing * 32 ? tops[i * MERGE_T + tid] : 0u;
      least = search(held, least, 2 * n);              // (its barriers come between these reads and what collect writes)
    }
    if (passing <= MERGE_LISTS) {
      for (int i = warp; i < passing; i += MERGE_WARPS) collect(s_list[i]);
    } else {
      for (int l = warp; l < lists; l += MERGE_WARPS)
        if (heads[l] >= least) collect(l);
    }
    if (ended)                                         // a beam that has ended stands for itself
      for (int k = tid; k < K; k += MERGE_T)
        if (ended[r * K + k] && isfinite(scores[r * K + k])) push((double)scores[r * K + k], 0.f, k * V + pad, -1 - k);
    __syncthreads();
    count = s_count;
    if (count <= MERGE_CAP || finer || !few) break;
    finer = true;
    __syncthreads();
    if (tid == 0) s_count = 0;
    __syncthreads();
  }
  auto value_of = [&](int e, int* index) {
    const int at = c_index[e];
    if (at < 0) {
      *index = (-1 - at) * V + pad;
      return (double)scores[r * K + -1 - at];
    }
    *index = at;
    return worth_of(at / V, c_value[e]);
  };
  int found = -1;
  if (count <= MERGE_CAP) {
    int ranked = count;
    if (count > MERGE_RANK) {
      // of many a second threshold, found the same way by the whole block
      unsigned held[MERGE_CAP / MERGE_T];
#pragma unroll
      for (int i = 0; i < MERGE_CAP / MERGE_T; i++) {
        int index;
        held[i] = i * MERGE_T + tid < count ? ordered((float)value_of(i * MERGE_T + tid, &index)) : 0u;
      }
      const unsigned low = search(held, 1u, MERGE_RANK);
      for (int e = tid; e < count; e += MERGE_T) {
        int index;
        const double a = value_of(e, &index);
        if (ordered((float)a) < low) continue;
        const int at = atomicAdd(&s_ranked, 1);
        if (at < MERGE_RANK) { s_value[at] = a; s_index[at] = index; }
      }
      __syncthreads();
      ranked = s_ranked;
    }
    if (ranked <= MERGE_RANK) {
      found = min(ranked, n);
      for (int e = tid; e < ranked; e += MERGE_T) {
        const double a = s_value[e];
        const int ai = s_index[e];
        int rank = 0;
        for (int i = 0; i < ranked; i++) rank += better(s_value[i], s_index[i], a, ai);
        if (rank < n) { s_out[rank] = a; s_out_at[rank] = ai; }
      }
    }
  }
  if (found < 0) {
    // more than there is room for (equal values): one after the other, each the best of what comes after the last.  The best of every 16th 512
    // tokens is known; the share that had the last is looked through again (480,000 equal values, 16 of them: 1.6 ms over all of them each
    // time, 0.55 this way).
    double last = INFINITY;
    int last_at = -1;
    auto best_of = [&](const double* value, const int* at, int of) {
      int x = 0;
      for (int w = 1; w < of; w++)
        if (better(value[w], at[w], value[x], at[x])) x = w;
      return x;
    };
    auto look = [&](int share) {
      double best = -INFINITY;
      int best_at = 0x7fffffff;
      auto take = [&](double a, int ai) {
        if (better(last, last_at, a, ai) && better(a, ai, best, best_at)) { best = a; best_at = ai; }
      };
      for (int k = 0; k < K; k++) {
        if (!s_alive[k]) continue;
        const float* const x = logits + (size_t)(r * K + k) * ld;
#pragma unroll 4
        for (int i = share * MERGE_T + tid; i < V; i += SHARES * MERGE_T) {
          const float f = x[i];
          if (f > -INFINITY) take(worth_of(k, f), k * V + i);
        }
      }
      if (ended && share == 0)
        for (int k = tid; k < K; k += MERGE_T)
          if (ended[r * K + k] && isfinite(scores[r * K + k])) take((double)scores[r * K + k], k * V + pad);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double f = __shfl_xor_sync(0xffffffffu, best, o);
        const int at = __shfl_xor_sync(0xffffffffu, best_at, o);
        if (better(f, at, best, best_at)) { best = f; best_at = at; }
      }
      if (lane == 0) { s_best[warp] = best; s_at[warp] = best_at; }
      __syncthreads();
      if (tid == 0) {
        const int x = best_of(s_best, s_at, MERGE_WARPS);
        s_share[share] = s_best[x];
        s_share_at[share] = s_at[x];
      }
      __syncthreads();
    };
    for (int share = 0; share < SHARES; share++) look(share);
    for (found = 0; found < n; found++) {
      const int x = best_of(s_share, s_share_at, SHARES);
      last = s_share[x];
      last_at = s_share_at[x];
      __syncthreads();
      if (last == -INFINITY) break;
      if (tid == 0) { s_out[found] = last; s_out_at[found] = last_at; }
      look(x);
    }
  }
  __syncthreads();
  if (tid == 0) {
    // fewer candidates than wanted: the first pairs that are none, of value -infinity
    int next = 0;
    for (int i = found; i < n; i++) {
      for (bool again = true; again;) {
        again = false;
        for (int j = 0; j < found; j++)
          if (s_out_at[j] == next) { next++; again = true; }
      }
      s_out[i] = -INFINITY;
      s_out_at[i] = next++;
    }
    if (placed) {                                      // (n == K) a beam's first child stays in its place, the others fill the rest
      unsigned long long used = 0, first = 0;
      for (int i = 0; i < n; i++) {
        const int k = s_out_at[i] / V;
        if (!(used >> k & 1)) { used |= 1ull << k; first |= 1ull << i; s_index[i] = k; }
      }
      int free_at = 0;
      for (int i = 0; i < n; i++) {
        if (first >> i & 1) continue;
        while (used >> free_at & 1) free_at++;
        used |= 1ull << free_at;
        s_index[i] = free_at;
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < n; i += MERGE_T) {
    const size_t to = (size_t)r * n + (placed ? s_index[i] : i);
    tokens[to] = s_out_at[i] % V;
    parents[to] = s_out_at[i] / V;
    out_scores[to] = (float)s_out[i];
  }
}

// ---- beams that go on from another one -----------------------------------------------------------------------
// A list of copies that read and write the same places: every thread has its part of all sources in registers before it
// writes, and parts are disjoint, so any map of beams to parents will do, cycles and several children of one parent included.
struct Move { long long from, to; int bytes; };        // byte offsets; how many bytes are to be taken over

// Pieces of Vec of every move, U of a thread at a time, `step` bytes apart, up to `end` and as far as a move consists of whole
// pieces of `whole` bytes.
template <typename Vec, int N, int U>
__device__ __forceinline__ void copy_held(char* base, const Move* moves, int count, long long at, int step, int end, int whole) {
  Vec v[U][N];
  auto in = [&](int u, int i) { return i < count && at + (long long)u * step + (int)sizeof(Vec) <= min(moves[i].bytes / whole * whole, end); };
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int i = 0; i < N; i++)
      if (in(u, i)) v[u][i] = __ldcs(reinterpret_cast<const Vec*>(base + moves[i].from + at + (long long)u * step));
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int i = 0; i < N; i++)
      if (in(u, i)) __stcs(reinterpret_cast<Vec*>(base + moves[i].to + at + (long long)u * step), v[u][i]);
}

constexpr int CP_T = 256, CP_BYTES = 16384;            // threads of a block, and the part of a row that it takes

// The block's part [lo, hi) of every move of the list, in pieces of Vec, and what a move has behind its last whole piece (pages with rows
// of odd sizes) in pieces of Unit.
template <typename Vec, typename Unit>
__device__ __forceinline__ void copy_part(char* base, const Move* moves, int count, int lo, int hi) {
  constexpr int W = (int)sizeof(Vec), PER = W / (int)sizeof(Unit);
  constexpr int MOST = PER > 1 ? (MAX_BEAMS * PER + CP_T - 1) / CP_T : 1;
  const int tid = threadIdx.x;
  Unit rest[MOST];
  auto rest_at = [&](int j) {                          // where the thread's j-th unit behind a move's whole pieces is, -1: nowhere
    const int e = tid + j * CP_T, i = e / PER;
    if (i >= count) return -1;
    const int at = moves[i].bytes / W * W + e % PER * (int)sizeof(Unit);
    return at >= lo && at < hi && at < moves[i].bytes ? at : -1;
  };
  if constexpr (PER > 1) {
#pragma unroll
    for (int j = 0; j < MOST; j++) {
      const int at = rest_at(j);
      if (at >= 0) rest[j] = *reinterpret_cast<const Unit*>(base + moves[(tid + j * CP_T) / PER].from + at);
    }
    __syncthreads();
  }
  if (count <= 2) {
    for (int at = lo + tid * W; at < hi; at += CP_T * W * 4) copy_held<Vec, 2, 4>(base, moves, count, at, CP_T * W, hi, W);
  } else if (count <= 4) {
    for (int at = lo + tid * W; at < hi; at += CP_T * W * 4) copy_held<Vec, 4, 4>(base, moves, count, at, CP_T * W, hi, W);
  } else if (count <= 16) {
    for (int at = lo + tid * W; at < hi; at += CP_T * W) copy_held<Vec, 16, 1>(base, moves, count, at, CP_T * W, hi, W);
  } else {                                             // many moves: a word of each in registers
    using Word = typename std::conditional<(W < 4), Vec, unsigned>::type;
    constexpr int S = (int)sizeof(Word);
    for (int at = lo + tid * S; at < hi; at += CP_T * S) copy_held<Word, MAX_BEAMS, 1>(base, moves, count, at, CP_T * S, hi, W);
  }
  if constexpr (PER > 1) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < MOST; j++) {
      const int at = rest_at(j);
      if (at >= 0) *reinterpret_cast<Unit*>(base + moves[(tid + j * CP_T) / PER].to + at) = rest[j];
    }
  }
}

// grid (parts of a slot's state, requests, layers).  Bound by HBM: 16 moved states of 6 layers of 3 MB, 604 MB in and out in 102 us (5.9 TB/s).
template <typename Vec>
__global__ void __launch_bounds__(CP_T)
beam_states_kernel(char* state, long long layer_bytes, long long slot_bytes, int bytes, int n_slots, const int* __restrict__ slots,
                   const int* __restrict__ parents, int K) {
  tlc_wait(state, slots, parents);
  __shared__ Move s_moves[MAX_BEAMS];
  __shared__ int s_count;
  const int r = blockIdx.y;
  if (threadIdx.x < 32) {
    int n = 0;
    for (int k0 = 0; k0 < K; k0 += 32) {
      const int k = k0 + threadIdx.x;
      int s = -1, from = -1;
      if (k < K) {
        const int p = parents[r * K + k];
        s = slots[r * K + k];
        if (p >= 0 && p < K && p != k) from = slots[r * K + p];
      }
      const bool move = s >= 0 && s < n_slots && from >= 0 && from < n_slots && from != s;
      const unsigned who = __ballot_sync(0xffffffffu, move);
      if (move) s_moves[n + __popc(who & ((1u << threadIdx.x) - 1))] = Move{from * slot_bytes, s * slot_bytes, bytes};
      n += __popc(who);
    }
    if (threadIdx.x == 0) s_count = n;
  }
  __syncthreads();
  if (s_count == 0) return;
  const long long lo = (long long)blockIdx.x * CP_BYTES;
  copy_part<Vec, Vec>(state + blockIdx.z * layer_bytes, s_moves, s_count, (int)lo, (int)min((long long)bytes, lo + CP_BYTES));
}

// A block a request.  Whole pages of the parent are shared; the page that the parent is filling is copied into the beam's own last
// page.  Where that page is whole and a child of the beam takes it over (lengths that differ: beam 0 of 64 positions goes on from beam 1 of 100,
// and beam 1 from beam 0), the copy goes into another page, one that the request's beams give back: the last page of a beam that fills none itself
// and that no child takes over.  Such beams take these pages in order; where there are too few the request is refused.
// own [R, K]: what the copy needs: {page it comes from, page it goes to, positions}.
constexpr int RO_T = 256, RO_COLS = 64;
enum { RO_LENGTH = 2, RO_SLOT = 3, RO_TABLE = 4, RO_SHARED = 5 };   // codes of the status word, as of page_resize
__global__ void __launch_bounds__(RO_T)
beam_tables_kernel(int* block_table, int n_slots, int max_pages, int* refs, int n_pages, int* lengths, const int* __restrict__ slots,
                   const int* __restrict__ parents, int K, int4* __restrict__ own, int* status) {
  tlc_wait(block_table, refs, lengths, slots, parents, own, status);
  __shared__ int s_slot[MAX_BEAMS], s_parent[MAX_BEAMS], s_len[MAX_BEAMS], s_last[MAX_BEAMS], s_fill[MAX_BEAMS], s_tile[MAX_BEAMS][RO_COLS], s_bad, s_cols;
  __shared__ unsigned char s_lost[MAX_BEAMS], s_spare[MAX_BEAMS];
  const int r = blockIdx.x, tid = threadIdx.x;
  if (tid == 0) s_bad = s_cols = 0;
  auto pages_of = [](int n) { return (int)(((unsigned)n + (TLC_PAGE - 1)) / TLC_PAGE); };      // (of a length up to 2^31 - 1)
  __syncthreads();
  if (tid < K) {
    const int s = slots[r * K + tid], p = parents[r * K + tid];
    s_slot[tid] = s;
    s_parent[tid] = p >= 0 && p < K ? p : tid;         // (a parent that is none: the beam stays as it is)
    const int n = s >= 0 && s < n_slots ? lengths[s] : 0;
    s_len[tid] = n;
    if (s >= n_slots || n < 0 || pages_of(n) > max_pages) atomicMax(&s_bad, s >= n_slots ? (int)RO_SLOT : (int)RO_LENGTH);
  }
  __syncthreads();
  if (tid < K && s_slot[tid] >= 0) {
    for (int k = 0; k < K; k++)
      if (k != tid && s_slot[k] == s_slot[tid]) atomicMax(&s_bad, (int)RO_SLOT);
    if (s_parent[tid] != tid && s_slot[s_parent[tid]] < 0) atomicMax(&s_bad, (int)RO_SLOT);
  }
  const int moved = __syncthreads_or(tid < K && s_parent[tid] != tid && s_slot[tid] >= 0), bad = s_bad;
  __syncthreads();
  if (bad == 0 && moved) {
    // the beams' own last pages, and how many columns there are to look at
    int count = 0;
    bool moves = false, fills = false;
    if (tid < K && s_slot[tid] >= 0) {
      const int have = pages_of(s_len[tid]), p = s_parent[tid];
      const int last = have > 0 ? block_table[(size_t)s_slot[tid] * max_pages + have - 1] : -1;
      const bool there = last >= 0 && last < n_pages;
      s_last[tid] = s_fill[tid] = last;
      atomicMax(&s_cols, have);
      if (p != tid) {
        count = there ? refs[last] : 0;
        fills = s_len[p] % TLC_PAGE != 0;
        if (fills && count != 1) atomicMax(&s_bad, count < 1 ? (int)RO_TABLE : (int)RO_SHARED);
      }
      moves = p != tid;
    }
    __syncthreads();
    // every entry that is going to be used names a page (64 rows of 2^25 entries are 2^31)
    for (unsigned e = tid, n = (unsigned)s_cols; e < K * n; e += RO_T) {
      const int k = (int)(e / n), c = (int)(e % n);
      if (s_slot[k] < 0 || c >= pages_of(s_len[k])) continue;
      const int page = block_table[(size_t)s_slot[k] * max_pages + c];
      if (page < 0 || page >= n_pages) atomicMax(&s_bad, (int)RO_TABLE);
    }
    const bool whole = tid < K && s_len[tid] % TLC_PAGE == 0;
    if (__syncthreads_or(fills && whole) && s_bad == 0) {
      // s_lost: the beam's last page goes to a child, and it fills one; s_spare: its last page is nobody's after the move
      if (tid < K) {
        bool taken = false;
        if (whole)
          for (int k = 0; k < K; k++) taken |= k != tid && s_parent[k] == tid && s_slot[k] >= 0;
        s_lost[tid] = fills && taken;
        s_spare[tid] = moves && !fills && !taken && s_len[tid] > 0 && count == 1;
      }
      __syncthreads();
      if (tid < K && s_lost[tid]) {
        int before = 0, at = 0;
        for (int k = 0; k < tid; k++) before += s_lost[k];
        for (; at < K; at++)
          if (s_spare[at] && before-- == 0) break;
        if (at < K) s_fill[tid] = s_last[at]; else atomicMax(&s_bad, (int)RO_SHARED);
      }
    }
  }
  __syncthreads();
  const bool go = s_bad == 0 && moved;
  if (tid < K) {
    const int p = s_parent[tid], used = s_len[p] % TLC_PAGE;
    int4 mv = make_int4(0, 0, 0, 0);
    if (go && p != tid && s_slot[tid] >= 0 && used > 0) mv = make_int4(s_last[p], s_fill[tid], used, 0);
    own[r * K + tid] = mv;
    if (go && p != tid && s_slot[tid] >= 0) lengths[s_slot[tid]] = s_len[p];
  }
  if (s_bad && tid == 0) atomicMax(status, s_bad);
  if (!go) return;
  const int cols = s_cols;
  for (int c0 = 0; c0 < cols; c0 += RO_COLS) {
    for (int e = tid; e < K * RO_COLS; e += RO_T) {
      const int k = e / RO_COLS, c = c0 + e % RO_COLS;
      if (s_slot[k] >= 0 && c < pages_of(s_len[k])) s_tile[k][e % RO_COLS] = block_table[(size_t)s_slot[k] * max_pages + c];
    }
    __syncthreads();
    // what is taken is counted before what is given back: a page that stays in use is never seen as somebody's alone by another request's block
    for (int give = 0; give < 2; give++) {
      for (int e = tid; e < K * RO_COLS; e += RO_T) {
        const int k = e / RO_COLS, i = e % RO_COLS, c = c0 + i, p = s_parent[k];
        if (p == k || s_slot[k] < 0) continue;
        const int have = pages_of(s_len[k]), full = s_len[p] / TLC_PAGE, used = s_len[p] % TLC_PAGE;
        const bool had = c < have, other = s_fill[k] != s_last[k];
        const bool keeps = used > 0 && c == have - 1 && !other;          // the page stays the beam's, in its new last place
        const int before = had ? s_tile[k][i] : -1;
        int after = 0;
        if (c < full) after = s_tile[p][i];
        else if (c == full && used > 0) after = s_fill[k];
        if (!had && c > full) continue;
        if (!give) {
          if (c < full ? !(had && !keeps && before == after) : c == full && used > 0 && other) atomicAdd(refs + after, 1);
        } else {
          if (had && !keeps && !(c < full && before == after)) atomicSub(refs + before, 1);
          if (c < full || had || (c == full && used > 0)) block_table[(size_t)s_slot[k] * max_pages + c] = after;
        }
      }
      __syncthreads();
    }
  }
}

// grid (parts of a page's positions of one head, requests, layers * heads of keys, then of values)
template <typename Unit>
__global__ void __launch_bounds__(CP_T)
beam_pages_kernel(char* k_pages, char* v_pages, long long layer_bytes, int KV, int row_bytes, int L, const int4* __restrict__ own, int K) {
  tlc_wait(k_pages, v_pages, own);
  __shared__ Move s_moves[MAX_BEAMS];
  __shared__ int s_count;
  const int r = blockIdx.y, region = TLC_PAGE * row_bytes;              // bytes of a head's positions in a page
  const int g = blockIdx.z % KV, l = blockIdx.z / KV % L;
  char* const base = (blockIdx.z >= (unsigned)(KV * L) ? v_pages : k_pages) + l * layer_bytes;
  if (threadIdx.x < 32) {
    int n = 0;
    for (int k0 = 0; k0 < K; k0 += 32) {
      const int k = k0 + threadIdx.x;
      const int4 mv = k < K ? own[r * K + k] : make_int4(0, 0, 0, 0);
      const unsigned who = __ballot_sync(0xffffffffu, mv.z > 0);
      if (mv.z > 0)
        s_moves[n + __popc(who & ((1u << threadIdx.x) - 1))] =
            Move{((long long)mv.x * KV + g) * region, ((long long)mv.y * KV + g) * region, mv.z * row_bytes};
      n += __popc(who);
    }
    if (threadIdx.x == 0) s_count = n;
  }
  __syncthreads();
  if (s_count == 0) return;
  const int lo = blockIdx.x * CP_BYTES;
  copy_part<uint4, Unit>(base, s_moves, s_count, lo, min(region, lo + CP_BYTES));
}

}  // namespace

// values of a piece: 64 a lane make few lists of long pieces; 16 spread a few rows over the SMs (4 rows of 65,536: 512 warps, not 128)
static int piece_values(long long rows, int V) { return rows * V >= 2048ll * 4 * tlc_sm_count() ? 2048 : 512; }

extern "C" long long tlc_beam_select_scratch(int rows, int V) {
  const int per = piece_values(rows, V);
  return rows * (((long long)V + per - 1) / per) * (long long)sizeof(Stats);
}

namespace {
struct SelectArgs {
  const float* logits;
  long long ld;
  const float* scores;
  const unsigned char* ended;
  int R, K, V, pieces, n, pad, placed;
  Stats* stats;
  int *tokens, *parents;
  float* out_scores;
};
template <int VPL, int VEC> int run_select(const SelectArgs& a, cudaStream_t stream) {
  static OncePerDevice ready;
  if (!ready.done([] {
        return cudaFuncSetAttribute(beam_merge_kernel<VPL, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (2 * MERGE_CAP + MAX_LISTS) * (int)sizeof(int));
      }))
    return tlc_fail(-2, "beam_select: cannot reserve shared memory");
  const unsigned blocks = (unsigned)(((long long)a.R * a.K * a.pieces + SCAN_WARPS - 1) / SCAN_WARPS);
  tlc_launch(beam_scan_kernel<VPL, VEC>, dim3(blocks), dim3(SCAN_WARPS * 32), 0, stream, a.logits, a.ld, a.scores, a.ended, a.R * a.K, a.V, a.pieces,
             a.stats);
  TLC_CHECK_LAUNCH("beam_select(scan)");
  tlc_launch(beam_merge_kernel<VPL, VEC>, dim3(a.R), dim3(MERGE_T), (2 * MERGE_CAP + (size_t)a.K * a.pieces) * sizeof(int), stream, a.logits, a.ld, a.scores,
             a.ended, a.K, a.V, a.pieces, a.n, a.pad, a.placed, a.stats, a.tokens, a.parents, a.out_scores);
  TLC_CHECK_LAUNCH("beam_select(merge)");
  return 0;
}
}  // namespace

extern "C" int tlc_beam_select(const float* logits, long long ld, const float* scores, const void* ended, int R, int K, int V, int n, int pad,
                               int placed, void* scratch, int* tokens, int* parents, float* out_scores, cudaStream_t stream) {
  if (R == 0) return 0;
  TLC_REQUIRE(R > 0 && R <= 65535 && K > 0 && K <= MAX_BEAMS && V > 0 && n > 0 && n <= MAX_N && n <= (long long)K * V,
              "beam_select: %d requests of %d beams (at most %d), %d candidates (at most %d) of %d tokens", R, K, MAX_BEAMS, n, MAX_N, V);
  TLC_REQUIRE(!placed || n == K, "beam_select: children take the beams' places where there are as many as beams, not %d for %d", n, K);
  TLC_REQUIRE(pad >= 0 && pad < V, "beam_select: token %d of %d", pad, V);
  const int per = piece_values((long long)R * K, V), pieces = (int)(((long long)V + per - 1) / per);
  TLC_REQUIRE((long long)K * pieces <= MAX_LISTS && (long long)K * V < (1ll << 31), "beam_select: %d beams of %d tokens are too many", K, V);
  TLC_REQUIRE((long long)R * K * pieces < (1ll << 31) * SCAN_WARPS, "beam_select: %d rows of %d logits are too many", R * K, V);
  TLC_REQUIRE(((uintptr_t)scratch & 15) == 0, "beam_select: scratch must start on a 16-byte boundary");
  const SelectArgs a{logits, ld, scores, (const unsigned char*)ended, R, K, V, pieces, n, pad, placed, (Stats*)scratch, tokens, parents, out_scores};
  const bool vec = ((uintptr_t)logits & 15) == 0 && ld % 4 == 0;
  if (per == 2048) return vec ? run_select<64, 4>(a, stream) : run_select<64, 1>(a, stream);
  return vec ? run_select<16, 4>(a, stream) : run_select<16, 1>(a, stream);
}

extern "C" int tlc_beam_reorder_states(void* state, long long layer_bytes, long long slot_bytes, long long bytes, int L, int n_slots,
                                       const int* slots, const int* parents, int R, int K, cudaStream_t stream) {
  if (R == 0 || L == 0 || bytes == 0) return 0;
  TLC_REQUIRE(R > 0 && R <= 65535 && K > 0 && K <= MAX_BEAMS && L > 0 && L <= 65535 && n_slots > 0 && bytes > 0 && bytes < (1ll << 31) - CP_BYTES,
              "beam_reorder_states: %d requests of %d beams (at most %d), %d layers of %lld bytes a slot", R, K, MAX_BEAMS, L, bytes);
  const long long all = (long long)(uintptr_t)state | layer_bytes | slot_bytes | bytes;
  const dim3 grid((unsigned)((bytes + CP_BYTES - 1) / CP_BYTES), R, L), block(CP_T);
  auto* const k = all % 16 == 0 ? beam_states_kernel<uint4> : all % 4 == 0 ? beam_states_kernel<unsigned> : all % 2 == 0 ? beam_states_kernel<unsigned short>
                                                                                                                 : beam_states_kernel<unsigned char>;
  tlc_launch(k, grid, block, 0, stream, (char*)state, layer_bytes, slot_bytes, (int)bytes, n_slots, slots, parents, K);
  TLC_CHECK_LAUNCH("beam_reorder_states");
  return 0;
}

extern "C" int tlc_beam_reorder_pages(int* block_table, int n_slots, int max_pages, int* refs, int n_pages, int* lengths, const int* slots,
                                      const int* parents, int R, int K, void* k_pages, void* v_pages, int dtype, int L, int KV, int hd,
                                      void* scratch, int* status, cudaStream_t stream) {
  if (R == 0) return 0;
  TLC_REQUIRE(R > 0 && R <= 65535 && K > 0 && K <= MAX_BEAMS, "beam_reorder_pages: %d requests of %d beams (at most %d)", R, K, MAX_BEAMS);
  TLC_REQUIRE(n_slots > 0 && max_pages > 0 && n_pages > 0 && n_pages <= (1 << 25) && L >= 0 && KV > 0 && hd > 0 && 2ll * L * KV <= 65535 && hd <= (1 << 20),
              "beam_reorder_pages: %d slots of %d pages, %d pages, %d layers of %d heads of %d", n_slots, max_pages, n_pages, L, KV, hd);
  TLC_REQUIRE(dtype == TLC_F32 || dtype == TLC_BF16, "unknown dtype code %d", dtype);
  TLC_REQUIRE((((uintptr_t)scratch | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0, "beam_reorder_pages: pages and scratch must start on 16-byte boundaries");
  tlc_launch(beam_tables_kernel, dim3(R), dim3(RO_T), 0, stream, block_table, n_slots, max_pages, refs, n_pages, lengths, slots, parents, K,
             (int4*)scratch, status);
  TLC_CHECK_LAUNCH("beam_reorder_pages(tables)");
  if (L == 0) return 0;
  const int row_bytes = hd * (dtype == TLC_F32 ? 4 : 2), region = TLC_PAGE * row_bytes;
  const dim3 grid((region + CP_BYTES - 1) / CP_BYTES, R, L * KV * (v_pages ? 2 : 1)), block(CP_T);
  auto* const k = row_bytes % 16 == 0 ? beam_pages_kernel<uint4> : beam_pages_kernel<unsigned short>;
  tlc_launch(k, grid, block, 0, stream, (char*)k_pages, (char*)v_pages, (long long)n_pages * KV * region, KV, row_bytes, L, (const int4*)scratch, K);
  TLC_CHECK_LAUNCH("beam_reorder_pages(copy)");
  return 0;
}
