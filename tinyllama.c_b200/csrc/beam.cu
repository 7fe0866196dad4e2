// Beam search on the GPU: the best candidates over beams and vocabulary, and beams that go on from another beam's keys, values and
// states.
//
// CodeClaper/tinyllama.c samples one sequence's next token on the host (sampler.c:107-257) and has no search over several.
// A candidate is a pair of beam k and token v of a request, of value
//     c_kv = s_k + x_kv - log(sum_u exp x_ku),
// and the n best of a request's K * V are wanted, equal values by the lowest k * V + v.  Two kernels:
//   * beam_scan_kernel reads every logit once.  A warp takes a piece of a row, 64 (or 16) values a lane in registers, and leaves the
//     piece's maximum, its sum of exponentials and its n largest logits in order.  Nothing crosses warps.  Which values can be
//     among the n largest: those not below the n-th largest of the maxima of 128 groups (four a lane), which a bitwise search by
//     ballots finds; some n to 2n values pass and are ranked by counting.
//   * beam_merge_kernel, a block a request, makes the rows' logarithms of sums and takes the n best of all lists the same way.
// Bound by HBM for a batch (256 rows of 130,048 logits: 133 MB, 20 us of loads), by the two launches for one request.
// Arithmetic: sums of exponentials in 32 bits over 16 values at most, from there on, and of the piece's largest values, in
// 64 bits, as are the logarithm and the values that are compared; two candidates change places only where they are nearer than
// the 2^-24 or so that this leaves.
#include "common.cuh"
#include <type_traits>

namespace {

constexpr int MAX_N = 64;                // candidates of a request
constexpr int MAX_BEAMS = 64;
constexpr int GROUPS = 4;                // groups of a lane's values
constexpr int CAP = 128;                 // values of a piece that pass the threshold and are ranked side by side
constexpr int SCAN_WARPS = 4;
constexpr int MERGE_T = 512, MERGE_CAP = 1024;
constexpr int MAX_LISTS = 40960;

struct Stats { double sum; float max; int pad; };      // of a piece: sum exp(x - max) and max

// larger float <=> larger unsigned
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr unsigned ORD_NEG_INF = 0x007fffffu;          // ordered(-infinity)

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ bool alive(const float* scores, const unsigned char* ended, int row) {
  return isfinite(scores[row]) && !(ended && ended[row]);
}

// grid: pieces of all rows, SCAN_WARPS a block.  VPL values a lane; VEC 4: rows start on 16-byte boundaries.
template <int VPL, int VEC>
__global__ void __launch_bounds__(SCAN_WARPS * 32)
beam_scan_kernel(const float* __restrict__ logits, long long ld, const float* __restrict__ scores, const unsigned char* __restrict__ ended,
                 int rows, int V, int n_pieces, int n, Stats* __restrict__ stats, int2* __restrict__ cand) {
  asm volatile("griddepcontrol.launch_dependents;");
  tlc_wait(logits, scores, ended, stats, cand);
  __shared__ float2 s_buf[SCAN_WARPS][CAP];
  const int lane = threadIdx.x & 31;
  float2* const buf = s_buf[threadIdx.x >> 5];
  const long long piece = (long long)blockIdx.x * SCAN_WARPS + (threadIdx.x >> 5);
  const int row = (int)(piece / n_pieces), p = (int)(piece % n_pieces);
  if (row >= rows || !alive(scores, ended, row)) return;
  const int base = p * 32 * VPL;
  const float* const x = logits + (size_t)row * ld + base;
  const int left = V - base;                           // values of the row from here on
  float v[VPL];
#pragma unroll
  for (int q = 0; q < VPL; q += VEC) {
    const int at = (q / VEC * 32 + lane) * VEC;
    if constexpr (VEC == 4) {
      if (at + 4 <= left) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(x + at));
        v[q] = f.x; v[q + 1] = f.y; v[q + 2] = f.z; v[q + 3] = f.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) v[q + e] = at + e < left ? __ldcs(x + at + e) : -INFINITY;
      }
    } else v[q] = at < left ? __ldcs(x + at) : -INFINITY;
  }
  auto index_of = [&](int q) { return base + (q / VEC * 32 + lane) * VEC + q % VEC; };
  // the groups' maxima (a NaN is nobody's maximum; it shows in the sum)
  unsigned key[GROUPS];
  float m = -INFINITY;
#pragma unroll
  for (int g = 0; g < GROUPS; g++) {
    float a = -INFINITY;
#pragma unroll
    for (int q = 0; q < VPL / GROUPS; q++) a = fmaxf(a, v[g * (VPL / GROUPS) + q]);
    key[g] = ordered(a);
    m = fmaxf(m, a);
  }
  m = warp_max(m);
  // the n-th largest of the 128 maxima: its bits from the highest down (any threshold that exactly n reach will do)
  unsigned least = 0;
  for (int bit = 31; bit >= 0; bit--) {
    const unsigned trial = least | 1u << bit;
    int reach = 0;
#pragma unroll
    for (int g = 0; g < GROUPS; g++) reach += __popc(__ballot_sync(0xffffffffu, key[g] >= trial));
    if (reach >= n) least = trial;
    if (reach == n) break;
  }
  least = max(least, ORD_NEG_INF + 1);                 // values of -infinity are nobody's candidates
  // as a float, larger than every value that does not pass
  const float bar = __uint_as_float(least & 0x80000000u ? least & 0x7fffffffu : ~least);
  int count = 0;
#pragma unroll
  for (int q = 0; q < VPL; q++) {
    const bool in = v[q] >= bar;
    const unsigned who = __ballot_sync(0xffffffffu, in);
    if (who) {
      const int at = count + __popc(who & ((1u << lane) - 1));
      if (in && at < CAP) buf[at] = make_float2(v[q], __int_as_float(index_of(q)));
      count += __popc(who);
    }
  }
  // sums: the values that did not pass in 32 bits, group by group, the others in 64 (they are what a peaked row consists of)
  const float top = m == -INFINITY ? 0.f : m;
  double sum = 0.0;
#pragma unroll
  for (int g = 0; g < GROUPS; g++) {
    float a = 0.f;
#pragma unroll
    for (int q = 0; q < VPL / GROUPS; q++) {
      const float u = v[g * (VPL / GROUPS) + q];
      a += count <= CAP && u >= bar ? 0.f : ex2((u - top) * 1.4426950408889634f);
    }
    sum += (double)a;
  }
  __syncwarp();
  int2* const out = cand + (size_t)piece * n;
  if (count <= CAP) {
    for (int e = lane; e < count; e += 32) {
      const float2 mine = buf[e];
      const int idx = __float_as_int(mine.y);
      int rank = 0;
      for (int i = 0; i < count; i++) {
        const float2 o = buf[i];
        rank += o.x > mine.x || (o.x == mine.x && __float_as_int(o.y) < idx);
      }
      if (rank < n) out[rank] = make_int2(__float_as_int(mine.x), idx);
      sum += exp((double)mine.x - (double)top);
    }
    for (int e = count + lane; e < n; e += 32) out[e] = make_int2(0, -1);
  } else {
    // many equal values (or all of the largest in one group): one after the other, the best that comes after the last
    float last = INFINITY;
    int last_at = -1;
    for (int r = 0; r < n; r++) {
      float best = -INFINITY;
      int best_at = 0x7fffffff;
#pragma unroll
      for (int q = 0; q < VPL; q++) {
        const int idx = index_of(q);
        const bool after = v[q] < last || (v[q] == last && idx > last_at);
        if (after && v[q] > -INFINITY && (v[q] > best || (v[q] == best && idx < best_at))) { best = v[q]; best_at = idx; }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float f = __shfl_xor_sync(0xffffffffu, best, o);
        const int at = __shfl_xor_sync(0xffffffffu, best_at, o);
        if (f > best || (f == best && at < best_at)) { best = f; best_at = at; }
      }
      if (lane == 0) out[r] = best > -INFINITY ? make_int2(__float_as_int(best), best_at) : make_int2(0, -1);
      last = best;
      last_at = best_at;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) stats[piece] = Stats{sum, m, 0};
}

// Candidates by value, equal ones by index.
__device__ __forceinline__ bool better(double a, int ai, double b, int bi) { return a > b || (a == b && ai < bi); }

__global__ void __launch_bounds__(MERGE_T)
beam_merge_kernel(const float* __restrict__ scores, const unsigned char* __restrict__ ended, int K, int V, int n_pieces, int n, int pad,
                  int placed, const Stats* __restrict__ stats, const int2* __restrict__ cand, int* __restrict__ tokens,
                  int* __restrict__ parents, float* __restrict__ out_scores) {
  tlc_pdl(scores, ended, stats, cand, tokens, parents, out_scores);
  extern __shared__ unsigned heads[];                  // of every list: the value of its first candidate, as an ordered integer
  __shared__ double s_off[MAX_BEAMS], s_value[MERGE_CAP], s_best[MERGE_T / 32];
  __shared__ int s_index[MERGE_CAP], s_at[MERGE_T / 32], s_count, s_alive[MAX_BEAMS];
  __shared__ unsigned s_least;
  __shared__ double s_out[MAX_N];
  __shared__ int s_out_at[MAX_N];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, lists = K * n_pieces;
  if (tid == 0) s_count = 0;
  // what a row's logits are raised by: the beam's score less the logarithm of the row's sum
  for (int k = warp; k < K; k += MERGE_T / 32) {
    const int row = r * K + k;
    bool on = alive(scores, ended, row);
    double off = 0.0;
    if (on) {
      const Stats* st = stats + (size_t)row * n_pieces;
      float m = -INFINITY;
      for (int i = lane; i < n_pieces; i += 32) m = fmaxf(m, st[i].max);
      m = warp_max(m);
      double sum = 0.0;
      for (int i = lane; i < n_pieces; i += 32) {
        const Stats a = st[i];
        // (a piece of nothing but -infinity and NaN: its sum is 0 or NaN)
        sum += a.max == -INFINITY ? (a.sum != a.sum ? a.sum : 0.0) : a.sum * exp((double)a.max - (double)m);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      off = (double)scores[row] - ((double)m + log(sum));
      on = isfinite(off);                              // no candidates of a row with a NaN, an infinity or nothing in it
    }
    if (lane == 0) { s_off[k] = off; s_alive[k] = on; }
  }
  __syncthreads();
  auto key_of = [&](int k, int bits) { return ordered((float)(s_off[k] + (double)__int_as_float(bits))); };
  const int2* const mine = cand + (size_t)r * lists * n;
  for (int l = tid; l < lists; l += MERGE_T) {
    const int k = l / n_pieces;
    unsigned h = 0;
    if (s_alive[k]) {
      const int2 c = mine[(size_t)l * n];
      if (c.y >= 0) h = key_of(k, c.x);
    }
    heads[l] = h;
  }
  __syncthreads();
  // the n-th largest of the first candidates: nothing below it can be among the n best
  if (warp == 0) {
    unsigned least = 0;
    for (int bit = 31; bit >= 0; bit--) {
      const unsigned trial = least | 1u << bit;
      int reach = 0;
      for (int l = lane; l < lists; l += 32) reach += heads[l] >= trial;
      reach = __reduce_add_sync(0xffffffffu, reach);
      if (reach >= n) least = trial;
      if (reach == n) break;
    }
    if (lane == 0) s_least = max(least, 1u);
  }
  __syncthreads();
  const unsigned least = s_least;
  for (int l = tid; l < lists; l += MERGE_T) {
    if (heads[l] < least) continue;
    const int k = l / n_pieces;
    for (int i = 0; i < n; i++) {
      const int2 c = mine[(size_t)l * n + i];
      if (c.y < 0 || key_of(k, c.x) < least) break;
      const int at = atomicAdd(&s_count, 1);
      if (at < MERGE_CAP) { s_value[at] = s_off[k] + (double)__int_as_float(c.x); s_index[at] = k * V + c.y; }
    }
  }
  if (ended)                                           // a beam that has ended stands for itself
    for (int k = tid; k < K; k += MERGE_T)
      if (ended[r * K + k] && isfinite(scores[r * K + k])) {
        const int at = atomicAdd(&s_count, 1);
        if (at < MERGE_CAP) { s_value[at] = (double)scores[r * K + k]; s_index[at] = k * V + pad; }
      }
  __syncthreads();
  const int count = s_count;
  int found;
  if (count <= MERGE_CAP) {
    found = min(count, n);
    for (int e = tid; e < count; e += MERGE_T) {
      const double a = s_value[e];
      const int ai = s_index[e];
      int rank = 0;
      for (int i = 0; i < count; i++) rank += better(s_value[i], s_index[i], a, ai);
      if (rank < n) { s_out[rank] = a; s_out_at[rank] = ai; }
    }
  } else {
    // more than there is room for (equal values in many lists): one after the other
    double last = INFINITY;
    int last_at = -1;
    found = 0;
    for (; found < n; found++) {
      double best = -INFINITY;
      int best_at = 0x7fffffff;
      auto take = [&](double a, int ai) {
        if (better(last, last_at, a, ai) && better(a, ai, best, best_at)) { best = a; best_at = ai; }
      };
      for (int l = tid; l < lists; l += MERGE_T) {
        if (heads[l] < least) continue;
        const int k = l / n_pieces;
        for (int i = 0; i < n; i++) {
          const int2 c = mine[(size_t)l * n + i];
          if (c.y < 0) break;
          take(s_off[k] + (double)__int_as_float(c.x), k * V + c.y);
        }
      }
      if (ended)
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
      best = s_best[0];
      best_at = s_at[0];
      for (int w = 1; w < MERGE_T / 32; w++)
        if (better(s_best[w], s_at[w], best, best_at)) { best = s_best[w]; best_at = s_at[w]; }
      __syncthreads();
      if (best == -INFINITY) break;
      if (tid == 0) { s_out[found] = best; s_out_at[found] = best_at; }
      last = best;
      last_at = best_at;
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

// grid (parts of a slot's state, requests, layers)
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
// page.  own [R, K]: what the copy needs: {page it comes from, page it goes to, positions}.
constexpr int RO_T = 256, RO_COLS = 64;
enum { RO_LENGTH = 2, RO_SLOT = 3, RO_TABLE = 4, RO_SHARED = 5 };   // codes of the status word, as of page_resize
__global__ void __launch_bounds__(RO_T)
beam_tables_kernel(int* block_table, int n_slots, int max_pages, int* refs, int n_pages, int* lengths, const int* __restrict__ slots,
                   const int* __restrict__ parents, int K, int4* __restrict__ own, int* status) {
  tlc_wait(block_table, refs, lengths, slots, parents, own, status);
  __shared__ int s_slot[MAX_BEAMS], s_parent[MAX_BEAMS], s_len[MAX_BEAMS], s_last[MAX_BEAMS], s_tile[MAX_BEAMS][RO_COLS], s_bad, s_cols;
  const int r = blockIdx.x, tid = threadIdx.x;
  if (tid == 0) s_bad = s_cols = 0;
  __syncthreads();
  if (tid < K) {
    const int s = slots[r * K + tid], p = parents[r * K + tid];
    s_slot[tid] = s;
    s_parent[tid] = p >= 0 && p < K ? p : tid;         // (a parent that is none: the beam stays as it is)
    const int n = s >= 0 && s < n_slots ? lengths[s] : 0;
    s_len[tid] = n;
    if (s >= n_slots || n < 0 || (n + TLC_PAGE - 1) / TLC_PAGE > max_pages) atomicMax(&s_bad, s >= n_slots ? (int)RO_SLOT : (int)RO_LENGTH);
  }
  __syncthreads();
  auto pages_of = [](int n) { return (n + TLC_PAGE - 1) / TLC_PAGE; };
  if (tid < K && s_slot[tid] >= 0) {
    for (int k = 0; k < K; k++)
      if (k != tid && s_slot[k] == s_slot[tid]) atomicMax(&s_bad, (int)RO_SLOT);
    if (s_parent[tid] != tid && s_slot[s_parent[tid]] < 0) atomicMax(&s_bad, (int)RO_SLOT);
  }
  const int moved = __syncthreads_or(tid < K && s_parent[tid] != tid && s_slot[tid] >= 0), bad = s_bad;
  __syncthreads();
  if (bad == 0 && moved) {
    // the beams' own last pages, and how many columns there are to look at
    if (tid < K && s_slot[tid] >= 0) {
      const int have = pages_of(s_len[tid]), p = s_parent[tid];
      s_last[tid] = have > 0 ? block_table[(size_t)s_slot[tid] * max_pages + have - 1] : -1;
      atomicMax(&s_cols, have);
      if (p != tid && s_len[p] % TLC_PAGE != 0) {
        const int last = s_last[tid];
        if (last < 0 || last >= n_pages) atomicMax(&s_bad, (int)RO_TABLE);
        else if (refs[last] != 1) atomicMax(&s_bad, refs[last] < 1 ? (int)RO_TABLE : (int)RO_SHARED);
      }
    }
    __syncthreads();
    // every entry that is going to be used names a page
    for (int e = tid; e < K * s_cols; e += RO_T) {
      const int k = e / s_cols, c = e % s_cols;
      if (s_slot[k] < 0 || c >= pages_of(s_len[k])) continue;
      const int page = block_table[(size_t)s_slot[k] * max_pages + c];
      if (page < 0 || page >= n_pages) atomicMax(&s_bad, (int)RO_TABLE);
    }
  }
  __syncthreads();
  const bool go = s_bad == 0 && moved;
  if (tid < K) {
    const int p = s_parent[tid], used = s_len[p] % TLC_PAGE;
    int4 mv = make_int4(0, 0, 0, 0);
    if (go && p != tid && s_slot[tid] >= 0 && used > 0) mv = make_int4(s_last[p], s_last[tid], used, 0);
    own[r * K + tid] = mv;
    if (go && p != tid && s_slot[tid] >= 0) lengths[s_slot[tid]] = s_len[p];
  }
  if (s_bad && tid == 0) atomicMax(status, s_bad);
  if (!go) return;
  const int cols = s_cols;
  for (int c0 = 0; c0 < cols; c0 += RO_COLS) {
    __syncthreads();
    for (int e = tid; e < K * RO_COLS; e += RO_T) {
      const int k = e / RO_COLS, c = c0 + e % RO_COLS;
      if (s_slot[k] >= 0 && c < pages_of(s_len[k])) s_tile[k][e % RO_COLS] = block_table[(size_t)s_slot[k] * max_pages + c];
    }
    __syncthreads();
    for (int e = tid; e < K * RO_COLS; e += RO_T) {
      const int k = e / RO_COLS, i = e % RO_COLS, c = c0 + i, p = s_parent[k];
      if (p == k || s_slot[k] < 0) continue;
      const int have = pages_of(s_len[k]), full = s_len[p] / TLC_PAGE, used = s_len[p] % TLC_PAGE;
      const bool had = c < have, keeps = used > 0 && c == have - 1;      // keeps: the page stays the beam's, in its new last place
      const int before = had ? s_tile[k][i] : -1;
      int after = 0;
      if (c < full) after = s_tile[p][i];
      else if (c == full && used > 0) after = s_last[k];
      if (!had && c > full) continue;
      if (c < full && !(had && !keeps && before == after)) atomicAdd(refs + after, 1);
      if (had && !keeps && !(c < full && before == after)) atomicSub(refs + before, 1);
      if (c < full || had || (c == full && used > 0)) block_table[(size_t)s_slot[k] * max_pages + c] = after;
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
static int piece_values(long long rows, int V) { return rows * V >= 2048ll * 148 * 4 ? 2048 : 512; }

extern "C" long long tlc_beam_select_scratch(int rows, int V, int n) {
  const int per = piece_values(rows, V);
  return rows * (((long long)V + per - 1) / per) * ((long long)sizeof(Stats) + 8ll * n);
}

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
  Stats* const stats = (Stats*)scratch;
  int2* const cand = (int2*)(stats + (size_t)R * K * pieces);
  const bool vec = ((uintptr_t)logits & 15) == 0 && ld % 4 == 0;
  const dim3 grid((unsigned)(((long long)R * K * pieces + SCAN_WARPS - 1) / SCAN_WARPS)), block(SCAN_WARPS * 32);
  auto* const k = per == 2048 ? (vec ? beam_scan_kernel<64, 4> : beam_scan_kernel<64, 1>) : (vec ? beam_scan_kernel<16, 4> : beam_scan_kernel<16, 1>);
  tlc_launch(k, grid, block, 0, stream, logits, ld, scores, (const unsigned char*)ended, R * K, V, pieces, n, stats, cand);
  TLC_CHECK_LAUNCH("beam_select(scan)");
  const int smem = K * pieces * (int)sizeof(unsigned);
  if (smem > 16 * 1024 &&
      cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_LISTS * (int)sizeof(unsigned)) != cudaSuccess)
    return tlc_fail(-2, "beam_select: cannot reserve shared memory");
  tlc_launch(beam_merge_kernel, dim3(R), dim3(MERGE_T), (size_t)smem, stream, scores, (const unsigned char*)ended, K, V, pieces, n, pad, placed,
             stats, cand, tokens, parents, out_scores);
  TLC_CHECK_LAUNCH("beam_select(merge)");
  return 0;
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
