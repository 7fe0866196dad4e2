// Attention of drafted tokens (a tree per request) over the paged cache, and the kernel that adds up partial results.
//
// CodeClaper/tinyllama.c attends causally, one sequence at a time (cpu_op.c:1010-1062); speculative decoding is no part of it.  Row i
// of a request's drafts sees the request's context (positions 0 .. start - 1 in the pages) and those drafts whose bit its mask has:
//     o_i = sum_j p_ij v_j,   p_ij = exp(s_ij) / (sum_j exp(s_ij) [+ exp(sink)]),   s_ij = cap(scale q_i . k_j)
// with cap(s) = softcap tanh(s / softcap).  The drafts' keys and values are read where the projections left them: nothing of a draft
// is in the cache before it is accepted.  A row that sees nothing has o = 0.
//
// The kernel here serves 32 bits and every head size up to 256; bfloat16 heads of 64 and 128 with a scale above 0 and no cap above 1,024 have their own
// (tree_attention_tc.cu).  A block walks the tiles of 64 keys of its segments (see tree_attention.cuh) with 64 (or 16) pairs of a row and a head of the
// group at a time, running maximum and sum per pair, all in 32 bits: scores and products by register tiles of 4 x 4
// from shared memory.  Bound by the CUDA cores' FFMA rate for many pairs, by the tiles' way into shared memory for few
// (32 bits, 3 requests of up to 1,900 keys, heads of 80: 20 us, of which the first tile's way in, two tiles a block and the sums' way out;
// bfloat16 heads of 256, 2 x 30,000 keys, 16 drafts of 16 heads: 637 us, 25 TFLOP/s).
#include "tree_attention.cuh"

namespace {

constexpr int NT = 256, BN = TLC_PAGE;
constexpr float LOG2E = 1.4426950408889634f;

__host__ __device__ constexpr int padded(int hd) { return ((hd + 3) / 4) % 2 ? (hd + 3) / 4 * 4 : (hd + 3) / 4 * 4 + 4; }   // 16-byte rows, an odd number of pieces
__host__ __device__ constexpr int smem_floats(int hd, int rows) { return (rows + BN) * padded(hd) + BN * ((hd + 63) / 64 * 64) + rows * (BN + 4); }

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ bool finite4(float4 v) { return isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w); }

// RM rows of pairs a thread (16 RM a tile), NJ times 64 columns of values.
template <typename T, int RM, int NJ>
__global__ void __launch_bounds__(NT)
tree_attention_kernel(TreeArgs a) {
  asm volatile("griddepcontrol.launch_dependents;");
  tlc_wait(a.q, a.k_new, a.v_new, a.k_pages, a.v_pages, a.block_table, a.slots, a.start, a.cu, a.positions, a.mask, a.out, a.part_o, a.part_ml,
           a.splits);
  constexpr int ROWS = 16 * RM;
  extern __shared__ float4 tree_raw[];
  const int hd = a.hd, hp = padded(hd), hv = NJ * 64, G = a.G;
  float* const Q = reinterpret_cast<float*>(tree_raw);
  float* const K = Q + ROWS * hp;
  float* const V = K + BN * hp;
  float* const P = V + BN * hv;                            // [ROWS][BN + 4]
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const T* const q = reinterpret_cast<const T*>(a.q);
  const TreeTake take = tree_plan<NT>(a, blockIdx.x, reinterpret_cast<int*>(tree_raw));
  int b = take.b, item = take.item, kt0 = take.tile, todo = take.todo;
  TreeSeq s = take.s;
  const float scale2 = a.scale * LOG2E;
  for (bool first_segment = true; todo > 0; first_segment = false) {
    while (item >= a.KV * s.row_tiles) { item -= a.KV * s.row_tiles; s = tree_seq(a, ++b); }
    const int g = item / s.row_tiles, r0 = item % s.row_tiles * a.tile_rows;
    const int kt1 = min(s.key_tiles, kt0 + todo);
    const int pairs = min(a.tile_rows, s.n * G - r0);
    const int* const table = a.block_table + (size_t)(s.context_tiles > 0 ? a.slots[b] : 0) * a.max_pages;
    __syncthreads();                                        // the segment before has used its queries
    // the tile's queries
    for (int r = ty; r < ROWS; r += 16) {
      const int i = (r0 + r) / G, h = g * G + (r0 + r) % G;
      const T* const from = q + (size_t)(s.t0 + i) * a.ld_q + (size_t)h * hd;
      if (a.vec) {
        for (int d = tx * 4; d < hd; d += 64) *reinterpret_cast<float4*>(Q + r * hp + d) = r < pairs ? load4(from + d) : make_float4(0.f, 0.f, 0.f, 0.f);
      } else {
        for (int d = tx; d < hp; d += 16) Q[r * hp + d] = r < pairs && d < hd ? to_f32(from[d]) : 0.f;
      }
    }
    float m[RM], l[RM], o[RM][4 * NJ];
    int pos[RM];
#pragma unroll
    for (int u = 0; u < RM; u++) {
      m[u] = -INFINITY;
      l[u] = 0.f;
#pragma unroll
      for (int c = 0; c < 4 * NJ; c++) o[u][c] = 0.f;
      const int r = ty * RM + u;
      pos[u] = r < pairs ? a.positions[s.t0 + (r0 + r) / G] : 0;
    }
    for (int kt = kt0; kt < kt1; kt++) {
      const bool draft = kt >= s.context_tiles;
      const int base = draft ? (kt - s.context_tiles) * BN : (s.first_tile + kt) * BN;       // first key of the tile: a draft's index, or a position
      const int keys = min(BN, (draft ? s.n : s.context) - base);
      const T *kr, *vr;
      size_t ldk, ldv;
      bool there = true;
      if (draft) {
        kr = reinterpret_cast<const T*>(a.k_new) + (size_t)(s.t0 + base) * a.ld_k + (size_t)g * hd;
        vr = reinterpret_cast<const T*>(a.v_new) + (size_t)(s.t0 + base) * a.ld_v + (size_t)g * hd;
        ldk = a.ld_k;
        ldv = a.ld_v;
      } else {
        const int page = table[base / BN];
        there = page >= 0 && page < a.n_pages;              // (a page that is none reads as zeros)
        const size_t at = ((size_t)(there ? page : 0) * a.KV + g) * (size_t)(BN * hd);
        kr = reinterpret_cast<const T*>(a.k_pages) + at;
        vr = reinterpret_cast<const T*>(a.v_pages) + at;
        ldk = ldv = hd;
      }
      bool odd = false;                                     // a value that is no number must not reach rows that do not see it
      if (a.vec) {
        // all of a thread's loads, then its stores (heads above 128: keys first)
        constexpr int HALVES = NJ > 2 ? 2 : 1;
#pragma unroll
        for (int half = 0; half < HALVES; half++) {
          float4 kv[4][NJ], vv[4][NJ];
#pragma unroll
          for (int x = 0; x < 4; x++)
#pragma unroll
            for (int c = 0; c < NJ; c++) {
              const int r = ty + 16 * x, d = 64 * c + tx * 4;
              const bool in = there && r < keys && d < hd;
              if (HALVES == 1 || half == 0) kv[x][c] = in ? load4(kr + r * ldk + d) : make_float4(0.f, 0.f, 0.f, 0.f);
              if (HALVES == 1 || half == 1) vv[x][c] = in ? load4(vr + r * ldv + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
          if (half == 0) __syncthreads();                   // the tile before has been used
#pragma unroll
          for (int x = 0; x < 4; x++)
#pragma unroll
            for (int c = 0; c < NJ; c++) {
              const int r = ty + 16 * x, d = 64 * c + tx * 4;
              if ((HALVES == 1 || half == 0) && d < hd) *reinterpret_cast<float4*>(K + r * hp + d) = kv[x][c];
              if (HALVES == 1 || half == 1) {
                *reinterpret_cast<float4*>(V + r * hv + d) = vv[x][c];
                odd |= !finite4(vv[x][c]);
              }
            }
        }
      } else {
        __syncthreads();                                    // the tile before has been used
        for (int r = ty; r < BN; r += 16) {
          for (int d = tx; d < hp; d += 16) K[r * hp + d] = there && r < keys && d < hd ? to_f32(kr[r * ldk + d]) : 0.f;
          for (int d = tx; d < hv; d += 16) {
            const float v = there && r < keys && d < hd ? to_f32(vr[r * ldv + d]) : 0.f;
            V[r * hv + d] = v;
            odd |= !isfinite(v);
          }
        }
      }
      odd = __syncthreads_or(odd);
      float sc[RM][4];
#pragma unroll
      for (int u = 0; u < RM; u++)
#pragma unroll
        for (int j = 0; j < 4; j++) sc[u][j] = 0.f;
      for (int d = 0; d < hd; d += 4) {
        float4 qv[RM], kv[4];
#pragma unroll
        for (int u = 0; u < RM; u++) qv[u] = *reinterpret_cast<const float4*>(Q + (ty * RM + u) * hp + d);
#pragma unroll
        for (int j = 0; j < 4; j++) kv[j] = *reinterpret_cast<const float4*>(K + (tx + 16 * j) * hp + d);
#pragma unroll
        for (int u = 0; u < RM; u++)
#pragma unroll
          for (int j = 0; j < 4; j++)
            sc[u][j] = fmaf(qv[u].x, kv[j].x, fmaf(qv[u].y, kv[j].y, fmaf(qv[u].z, kv[j].z, fmaf(qv[u].w, kv[j].w, sc[u][j]))));
      }
#pragma unroll
      for (int u = 0; u < RM; u++) {
        const int r = ty * RM + u, i = (r0 + r) / G;
        float mx = m[u];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int key = tx + 16 * j;
          bool sees = r < pairs && key < keys;
          if (sees) sees = draft ? tree_sees(a, s.t0, i, base + key) : a.window <= 0 || base + key > pos[u] - a.window;
          float x = sc[u][j] * scale2;
          if (a.softcap > 0.f) x = a.softcap * LOG2E * tanhf(sc[u][j] * a.scale / a.softcap);
          sc[u][j] = sees ? x : -INFINITY;
          mx = fmaxf(mx, sc[u][j]);
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        const float ref = mx == -INFINITY ? 0.f : mx, shrink = m[u] == -INFINITY ? 0.f : exp2f(m[u] - ref);
        m[u] = mx;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float p = exp2f(sc[u][j] - ref);
          sum += p;
          P[r * (BN + 4) + tx + 16 * j] = p;
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        l[u] = (l[u] == 0.f ? 0.f : l[u] * shrink) + sum;
#pragma unroll
        for (int c = 0; c < 4 * NJ; c++) o[u][c] = o[u][c] == 0.f ? 0.f : o[u][c] * shrink;
      }
      __syncwarp();                                         // a row of P is written and read by the same 16 lanes
      if (!odd) {
        for (int k = 0; k < BN; k += 4) {
          float4 p[RM];
#pragma unroll
          for (int u = 0; u < RM; u++) p[u] = *reinterpret_cast<const float4*>(P + (ty * RM + u) * (BN + 4) + k);
#pragma unroll
          for (int x = 0; x < 4; x++)
#pragma unroll
            for (int c = 0; c < NJ; c++) {
              const float4 v = *reinterpret_cast<const float4*>(V + (k + x) * hv + 64 * c + tx * 4);
#pragma unroll
              for (int u = 0; u < RM; u++) {
                const float w = x == 0 ? p[u].x : x == 1 ? p[u].y : x == 2 ? p[u].z : p[u].w;
                o[u][4 * c] = fmaf(w, v.x, o[u][4 * c]);
                o[u][4 * c + 1] = fmaf(w, v.y, o[u][4 * c + 1]);
                o[u][4 * c + 2] = fmaf(w, v.z, o[u][4 * c + 2]);
                o[u][4 * c + 3] = fmaf(w, v.w, o[u][4 * c + 3]);
              }
            }
        }
      } else {
        for (int k = 0; k < BN; k++)
#pragma unroll
          for (int u = 0; u < RM; u++) {
            const float w = P[(ty * RM + u) * (BN + 4) + k];
            if (w == 0.f) continue;
#pragma unroll
            for (int c = 0; c < 4 * NJ; c++) o[u][c] = fmaf(w, V[k * hv + 64 * (c / 4) + tx * 4 + c % 4], o[u][c]);
          }
      }
    }
    const bool whole = kt0 == 0 && kt1 == s.key_tiles;
#pragma unroll
    for (int u = 0; u < RM; u++) {
      const int r = ty * RM + u;
      if (r >= pairs) continue;
      const int i = (r0 + r) / G, h = g * G + (r0 + r) % G;
      if (whole) {
        float total = l[u], mx = m[u];
        float f = 1.f;
        if (a.sink) {
          const float sv = a.sink_values ? a.sink_values[h] * LOG2E : 0.f, top = fmaxf(mx, sv);
          f = mx == -INFINITY && total == 0.f ? 0.f : exp2f(mx - top);
          total = (total == 0.f ? 0.f : total * f) + exp2f(sv - top);
        }
        const float inv = l[u] == 0.f ? 0.f : f / total;
        T* const to = reinterpret_cast<T*>(a.out) + (size_t)(s.t0 + i) * a.out_ld + (size_t)h * hd;
#pragma unroll
        for (int c = 0; c < 4 * NJ; c++) {
          const int d = 64 * (c / 4) + tx * 4 + c % 4;
          if (d < hd) to[d] = from_f32<T>(l[u] == 0.f ? 0.f : o[u][c] * inv);
        }
      } else {
        const int slot = first_segment ? 0 : 1;
        if (tx == 0) *tree_part_ml(a, blockIdx.x, slot, r) = make_float2(m[u], l[u]);
#pragma unroll
        for (int c = 0; c < NJ; c++)
          if (64 * c + tx * 4 < hd) *tree_part(a, blockIdx.x, slot, 16 * c + tx, r) = make_float4(o[u][4 * c], o[u][4 * c + 1], o[u][4 * c + 2], o[u][4 * c + 3]);
      }
    }
    todo -= kt1 - kt0;
    kt0 = 0;
    item++;
  }
}

__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
  const __nv_bfloat162 u[2] = {__floats2bfloat162_rn(v.x, v.y), __floats2bfloat162_rn(v.z, v.w)};
  *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(u);
}
// four columns from d on of a row of hd, times f
template <typename T> __device__ __forceinline__ void put4(const TreeArgs& a, T* row, int d, float4 v, float f, bool none) {
  v = none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
  if (a.vec_out) {
    if (d < a.hd) store4(row + d, v);
    return;
  }
  const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int q = 0; q < 4; q++)
    if (d + q < a.hd) row[d + q] = from_f32<T>(o[q]);
}

// Items that several blocks share: o = sum_z o_z 2^(m_z - m) / (sum_z l_z 2^(m_z - m) [+ 2^(sink - m)]).  Every block reads which items those
// are (an entry of splits for each block of the kernel before) and takes its share of their rows, four at a time, which lie side by
// side: of few rows in many segments a block, or one for some of the columns, the segments shared out over its warps, else a warp.  Bound by trips to
// the L2, of which rows take two (the statistics, then the values of some segments at a time); a launch with nothing to add up is over
// after one.
constexpr int MG_T = 256, MG_WARPS = MG_T / 32, MG_MOST = 512;           // MG_MOST: blocks of the kernel before, at most
constexpr int MG_ROWS = 4, MG_LANES = 32 / MG_ROWS;                      // rows of a task, lanes to a row
constexpr int MG_E = 2;                                                  // fours of columns of a lane where a warp has the task
template <typename T>
__global__ void __launch_bounds__(MG_T)
tree_merge_kernel(TreeArgs a) {
  tlc_pdl(a.part_o, a.part_ml, a.splits, a.out);
  __shared__ int s_before[MG_MOST], s_warp[MG_WARPS], s_most[MG_WARPS];
  __shared__ float s_w[MG_MOST][MG_ROWS], s_red[2 * MG_WARPS][MG_ROWS];
  __shared__ float4 s_acc[2][MG_WARPS][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = a.G, hd = a.hd;
  // the items' rows, in fours, and the most segments of an item
  constexpr int EACH = MG_MOST / MG_T;
  int total = 0, most = 0;
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const int c = i * MG_T + tid;
    if (i * MG_T >= a.blocks) {
      s_before[c] = 0x7fffffff;
      continue;
    }
    TreeSplit sp = {};
    if (c < a.blocks) sp = a.splits[c];
    const int n = sp.n > 1 ? (sp.pairs + MG_ROWS - 1) / MG_ROWS : 0;
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const int segments = __reduce_max_sync(0xffffffffu, sp.n);
    if (i > 0) __syncthreads();
    if (lane == 31) { s_warp[warp] = x; s_most[warp] = segments; }
    __syncthreads();
    int before = total + x - n;
#pragma unroll
    for (int w = 0; w < MG_WARPS; w++) {
      if (w < warp) before += s_warp[w];
      total += s_warp[w];
      most = max(most, s_most[w]);
    }
    s_before[c] = before;
  }
  if (total == 0) return;
  __syncthreads();
  auto task_of = [&](int at) {                             // the last block whose rows start at or before these
    int c = 0;
#pragma unroll
    for (int step = MG_MOST / 2; step > 0; step >>= 1)
      if (s_before[c + step] <= at) c += step;
    return c;
  };
  // what a task takes, in half trips to the L2: of a warp, which reads eight segments at a time, six and four for each eight; of a block, which has
  // eight warps do that, four and two or more for every 32 columns.  (4 x 60,000 keys, 2,048 rows in 19 segments: warps 88 us with the kernel before,
  // blocks 97; 60,000 keys, 512 rows in 74 segments: warps 57, blocks 40; 16 x 1,000 keys, 2,048 rows in 2 segments: warps 17, blocks 38; 45,000 and
  // 60,000 keys, 888 rows in 37 segments: warps 64, blocks 59.)
  const int grid = gridDim.x, wide = grid * MG_WARPS, chunks = (hd + 31) / 32, cuts = (hd + 32 * MG_E - 1) / (32 * MG_E);
  int parts = 0, trips = (total * cuts + wide - 1) / wide * (6 + (most + 7) / 8 * 4);  // parts: blocks that share a row's columns
  for (int p = chunks; p > 0; p = (p + 1) / 2) {
    const int t = (total * p + grid - 1) / grid * (4 + (chunks + p - 1) / p * (32 + most) / 16);
    if (t < trips) { trips = t; parts = p; }
    if (p == 1) break;
  }
  if (parts > 0) {
    // a lane has four columns of a row, 32 columns at a time, the warps have every eighth segment
    for (int at = blockIdx.x; at < total * parts; at += grid) {
      const int c = task_of(at / parts), per = (chunks + parts - 1) / parts, chunk0 = at % parts * per;
      const TreeSplit item = a.splits[c];
      const int n = item.n, r = (at / parts - s_before[c]) * MG_ROWS, row = r + lane % MG_ROWS, own = min(row, item.pairs - 1), h = item.g * G + (item.r0 + own) % G;
      auto stats = [&](int z) { return *tree_part_ml(a, item.c0 + z, z == 0 ? item.slot0 : 0, own); };
      // the statistics of the lane's row, every 64th segment a thread
      float2 ml[MG_MOST / (MG_T / MG_ROWS)];
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int i = 0; i < MG_MOST / (MG_T / MG_ROWS); i++) {
        const int z = i * (MG_T / MG_ROWS) + tid / MG_ROWS;
        ml[i] = z < n ? stats(z) : make_float2(-INFINITY, 0.f);
        if (ml[i].y != 0.f) m = fmaxf(m, ml[i].x);
      }
#pragma unroll
      for (int o = MG_ROWS; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      __syncthreads();                                     // the task before has been read
      if (lane < MG_ROWS) s_red[warp][lane] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < MG_WARPS; w++) m = fmaxf(m, s_red[w][lane % MG_ROWS]);
      const float sv = a.sink && a.sink_values ? a.sink_values[h] * LOG2E : 0.f;
      if (a.sink) m = fmaxf(m, sv);
#pragma unroll
      for (int i = 0; i < MG_MOST / (MG_T / MG_ROWS); i++) {
        const int z = i * (MG_T / MG_ROWS) + tid / MG_ROWS;
        if (z >= n) continue;
        const float w = ml[i].y != 0.f ? exp2f(ml[i].x - m) : 0.f;
        s_w[z][lane % MG_ROWS] = w;
        if (ml[i].y != 0.f) l += ml[i].y * w;
      }
#pragma unroll
      for (int o = MG_ROWS; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      if (lane < MG_ROWS) s_red[MG_WARPS + warp][lane] = l;
      __syncthreads();
      l = 0.f;
#pragma unroll
      for (int w = 0; w < MG_WARPS; w++) l += s_red[MG_WARPS + w][lane % MG_ROWS];
      const float inv = l == 0.f ? 0.f : 1.0f / (a.sink ? l + exp2f(sv - m) : l);
      T* const to = reinterpret_cast<T*>(a.out) + (size_t)(item.t0 + (item.r0 + own) / G) * a.out_ld + (size_t)h * hd;
      for (int part = chunk0; part < min(chunks, chunk0 + per); part++) {
        const int chunk = part * 8 + lane / MG_ROWS;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        constexpr int Z = 10;
        for (int z0 = warp; z0 < n; z0 += Z * MG_WARPS) {
          float4 v[Z];
#pragma unroll
          for (int i = 0; i < Z; i++) {
            const int z = min(z0 + i * MG_WARPS, n - 1);
            v[i] = *tree_part(a, item.c0 + z, z == 0 ? item.slot0 : 0, min(chunk, (hd + 3) / 4 - 1), own);
          }
#pragma unroll
          for (int i = 0; i < Z; i++) {
            const float w = z0 + i * MG_WARPS < n ? s_w[z0 + i * MG_WARPS][lane % MG_ROWS] : 0.f;
            if (w == 0.f) continue;
            sum.x = fmaf(v[i].x, w, sum.x);
            sum.y = fmaf(v[i].y, w, sum.y);
            sum.z = fmaf(v[i].z, w, sum.z);
            sum.w = fmaf(v[i].w, w, sum.w);
          }
        }
        float4 (*const room)[32] = s_acc[part & 1];        // (read while the next 32 columns' are written)
        room[warp][lane] = sum;
        __syncthreads();
        if (warp != part % MG_WARPS || row >= item.pairs) continue;
        sum = room[0][lane];
#pragma unroll
        for (int w = 1; w < MG_WARPS; w++) {
          const float4 o = room[w][lane];
          sum.x += o.x; sum.y += o.y; sum.z += o.z; sum.w += o.w;
        }
        put4(a, to, chunk * 4, sum, inv, l == 0.f);
      }
    }
    return;
  }
  for (int at = blockIdx.x * MG_WARPS + warp; at < total * cuts; at += wide) {
    const int c = task_of(at / cuts), chunk = at % cuts * (8 * MG_E) + lane / MG_ROWS, last = (hd + 3) / 4 - 1;
    const TreeSplit item = a.splits[c];
    const int n = item.n, row = (at / cuts - s_before[c]) * MG_ROWS + lane % MG_ROWS, own = min(row, item.pairs - 1), h = item.g * G + (item.r0 + own) % G;
    // a lane has every eighth four columns of a row, and the statistics of every eighth segment
    auto stats = [&](int z) { return z < n ? *tree_part_ml(a, item.c0 + z, z == 0 ? item.slot0 : 0, own) : make_float2(-INFINITY, 0.f); };
    const float sv = a.sink && a.sink_values ? a.sink_values[h] * LOG2E : 0.f;
    float2 ml = stats(lane / MG_ROWS);
    float m = ml.y != 0.f ? ml.x : -INFINITY, l = 0.f;
    for (int z = MG_LANES + lane / MG_ROWS; z < n; z += MG_LANES) {
      const float2 o = stats(z);
      if (o.y != 0.f) m = fmaxf(m, o.x);
    }
#pragma unroll
    for (int o = MG_ROWS; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (a.sink) m = fmaxf(m, sv);
    float4 acc[MG_E];
#pragma unroll
    for (int e = 0; e < MG_E; e++) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int base = 0; base < n; base += MG_LANES) {
      if (base > 0) ml = stats(base + lane / MG_ROWS);
      const float w = ml.y != 0.f ? exp2f(ml.x - m) : 0.f;
      if (ml.y != 0.f) l += ml.y * w;
      float4 v[MG_LANES][MG_E];                            // all eight segments on their way
#pragma unroll
      for (int z = 0; z < MG_LANES; z++) {
        if (base + z >= n) continue;
#pragma unroll
        for (int e = 0; e < MG_E; e++) v[z][e] = *tree_part(a, item.c0 + base + z, base + z == 0 ? item.slot0 : 0, min(chunk + 8 * e, last), own);
      }
#pragma unroll
      for (int z = 0; z < MG_LANES; z++) {
        const float wz = __shfl_sync(0xffffffffu, w, z * MG_ROWS + lane % MG_ROWS);
        if (base + z >= n || wz == 0.f) continue;
#pragma unroll
        for (int e = 0; e < MG_E; e++) {
          acc[e].x = fmaf(v[z][e].x, wz, acc[e].x);
          acc[e].y = fmaf(v[z][e].y, wz, acc[e].y);
          acc[e].z = fmaf(v[z][e].z, wz, acc[e].z);
          acc[e].w = fmaf(v[z][e].w, wz, acc[e].w);
        }
      }
    }
#pragma unroll
    for (int o = MG_ROWS; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const float inv = l == 0.f ? 0.f : 1.0f / (a.sink ? l + exp2f(sv - m) : l);
    if (row >= item.pairs) continue;
    T* const to = reinterpret_cast<T*>(a.out) + (size_t)(item.t0 + (item.r0 + row) / G) * a.out_ld + (size_t)h * hd;
#pragma unroll
    for (int e = 0; e < MG_E; e++) put4(a, to, (chunk + 8 * e) * 4, acc[e], inv, l == 0.f);
  }
}

template <typename T> void run_merge(const TreeArgs& a, cudaStream_t stream) {
  const long long tasks = ((long long)a.T * a.H + MG_ROWS - 1) / MG_ROWS * ((a.hd + 31) / 32), most = 2 * tlc_sm_count();     // two to an SM
  const dim3 grid((unsigned)(tasks < most ? tasks : most));
  tlc_launch(tree_merge_kernel<T>, grid, dim3(MG_T), 0, stream, a);
}

constexpr int SIMT_MOST_SMEM = 227 * 1024 - 1024;
static_assert(smem_floats(256, 64) * 4 <= SIMT_MOST_SMEM && (smem_floats(192, 64) + BN * 64) * 4 <= SIMT_MOST_SMEM, "shared memory of a block");
template <typename T, int RM> int run_simt(const TreeArgs& a, cudaStream_t stream) {
  const int nj = (a.hd + 63) / 64, smem = smem_floats(a.hd, 16 * RM) * (int)sizeof(float);
  auto* const k = nj == 1 ? tree_attention_kernel<T, RM, 1> : nj == 2 ? tree_attention_kernel<T, RM, 2> : tree_attention_kernel<T, RM, 4>;
  const int full = nj <= 2 ? smem : smem + BN * (256 - nj * 64) * (int)sizeof(float);
  static OncePerDevice ready[3];
  if (!ready[nj == 1 ? 0 : nj == 2 ? 1 : 2].done([&] { return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SIMT_MOST_SMEM); }))
    return tlc_fail(-2, "tree_attention: cannot reserve %d bytes of shared memory", full);
  tlc_launch(k, dim3(a.blocks), dim3(NT), (size_t)full, stream, a);
  TLC_CHECK_LAUNCH("tree_attention");
  return 0;
}

}  // namespace

int tlc_tree_attention_simt(const TreeArgs& a, int dtype, int rows, cudaStream_t stream) {
  TLC_DISPATCH_DTYPE(dtype, T, return rows == 64 ? (run_simt<T, 4>(a, stream)) : (run_simt<T, 1>(a, stream)));
}

// How a call is cut: by which kernel, pairs of a tile, blocks, and the scratch that it needs.
namespace {
struct Cut { bool tc; int rows, tile_rows, blocks; long long units, scratch; };
Cut cut_of(int dtype, int aligned, int n_pages, int B, int T, int H, int KV, int hd, int max_context, int max_new) {
  Cut c;
  const int G = H / KV;
  c.tc = tlc_tree_attention_tc_takes(dtype, aligned, H, KV, hd, n_pages);
  c.rows = c.tc ? 256 : (long long)max_new * G > 16 ? 64 : 16;
  c.tile_rows = c.tc ? 128 / G * G * 2 : c.rows;
  const long long kt = ((long long)max_context + BN - 1) / BN + (max_new + BN - 1) / BN;
  c.units = (((long long)T * G + c.tile_rows - 1) / c.tile_rows + B) * KV * kt;
  const long long wave = (long long)tlc_sm_count() * (c.tc ? 1 : 2);
  c.blocks = (int)(c.units < wave ? (c.units < 1 ? 1 : c.units) : wave);
  if (c.blocks > MG_MOST) c.blocks = MG_MOST;
  c.scratch = (long long)c.blocks * (2 * c.rows * ((hd + 3) / 4 * 4 + 2) * 4 + (long long)sizeof(TreeSplit));
  return c;
}
}  // namespace

extern "C" long long tlc_tree_attention_scratch(int dtype, int aligned, int n_pages, int B, int T, int H, int KV, int hd, int max_context, int max_new) {
  if (KV <= 0 || H <= 0 || H % KV) return 0;
  return cut_of(dtype, aligned, n_pages, B, T, H, KV, hd, max_context, max_new).scratch;
}

extern "C" int tlc_tree_attention(const void* q, int dtype, int ld_q, const void* k_new, int ld_k, const void* v_new, int ld_v, const void* k_pages,
                                  const void* v_pages, int n_pages, const int* block_table, int n_slots, int max_pages, const int* slots,
                                  const int* start, const int* cu_seqlens, const int* positions, const int* mask, int words, void* out,
                                  int out_ld, int B, int T, int H, int KV, int hd, float scale, int window, float softcap, int sink,
                                  const float* sink_values, int max_context, int max_new, void* scratch, int aligned, cudaStream_t stream) {
  if (B == 0 || T == 0) return 0;
  TLC_REQUIRE(B > 0 && T > 0 && KV > 0 && H > 0 && H % KV == 0 && H <= 65535 * 4 && hd >= 1 && hd <= 256,
              "tree_attention: %d rows of %d requests, %d heads over %d of size %d (at most 256)", T, B, H, KV, hd);
  TLC_REQUIRE(max_context >= 0 && max_new >= 0 && n_pages > 0 && n_slots > 0 && max_pages > 0 && (mask == nullptr || words > 0),
              "tree_attention: contexts of %d, %d new rows, %d pages", max_context, max_new, n_pages);
  TLC_REQUIRE(((uintptr_t)scratch & 15) == 0, "tree_attention: scratch must start on a 16-byte boundary");
  const Cut c = cut_of(dtype, aligned, n_pages, B, T, H, KV, hd, max_context, max_new);
  TLC_REQUIRE(!c.tc || (scale > 0.f && softcap <= 1024.f), "tree_attention: a scale of %g, scores capped at %g, with `aligned` set", (double)scale, (double)softcap);
  TLC_REQUIRE(c.units < (1ll << 31), "tree_attention: %d rows over %d keys are too many", T, max_context);
  TreeArgs a = {};
  a.q = q; a.k_new = k_new; a.v_new = v_new; a.k_pages = k_pages; a.v_pages = v_pages;
  a.ld_q = ld_q; a.ld_k = ld_k; a.ld_v = ld_v; a.n_pages = n_pages;
  a.block_table = block_table; a.slots = slots; a.start = start; a.cu = cu_seqlens; a.positions = positions; a.mask = mask;
  a.n_slots = n_slots; a.max_pages = max_pages; a.words = words;
  a.out = out; a.out_ld = out_ld; a.B = B; a.T = T; a.H = H; a.KV = KV; a.hd = hd;
  a.scale = scale; a.window = window > 0 ? window : 0; a.softcap = softcap; a.sink = sink; a.sink_values = sink_values;
  a.max_context = max_context; a.max_new = max_new;
  a.err = tlc_error_words_here();
  const uintptr_t starts = (uintptr_t)q | (uintptr_t)k_new | (uintptr_t)v_new | (uintptr_t)k_pages | (uintptr_t)v_pages;
  a.G = H / KV;
  a.vec_out = hd % 4 == 0 && (out_ld & 3) == 0 && ((uintptr_t)out & (dtype == TLC_F32 ? 15 : 7)) == 0;
  a.vec = hd % 4 == 0 && ((ld_q | ld_k | ld_v) & 3) == 0 && (starts & (dtype == TLC_F32 ? 15 : 7)) == 0;
  a.tile_rows = c.tile_rows;
  a.blocks = c.blocks;
  a.part_rows = c.rows;
  a.part_o = (float*)scratch;
  a.part_ml = a.part_o + (size_t)c.blocks * 2 * c.rows * ((hd + 3) / 4 * 4);
  a.splits = (TreeSplit*)(a.part_ml + (size_t)c.blocks * 2 * c.rows * 2);
  if (const int rc = c.tc ? tlc_tree_attention_tc(a, stream) : tlc_tree_attention_simt(a, dtype, c.rows, stream)) return rc;
  TLC_DISPATCH_DTYPE(dtype, E, run_merge<E>(a, stream));
  TLC_CHECK_LAUNCH("tree_attention(merge)");
  return 0;
}
