// Attention of drafted tokens (a tree per request) over the paged cache, and the kernel that adds up partial results.
//
// CodeClaper/tinyllama.c attends causally, one sequence at a time (cpu_op.c:1010-1062); speculative decoding is no part of it.  Row i
// of a request's drafts sees the request's context (positions 0 .. start - 1 in the pages) and those drafts whose bit its mask has:
//     o_i = sum_j p_ij v_j,   p_ij = exp(s_ij) / (sum_j exp(s_ij) [+ exp(sink)]),   s_ij = cap(scale q_i . k_j)
// with cap(s) = softcap tanh(s / softcap).  The drafts' keys and values are read where the projections left them: nothing of a draft
// is in the cache before it is accepted.  A row that sees nothing has o = 0.
//
// The kernel here serves 32 bits and every head size up to 256; bfloat16 heads of 64 and 128 have their own
// (tree_attention_tc.cu).  A block walks the tiles of 64 keys of its segments (see tree_attention.cuh) with 64 (or 16) pairs of a row and a head of the
// group at a time, running maximum and sum per pair, all in 32 bits: scores and products by register tiles of 4 x 4
// from shared memory.  Bound by the CUDA cores' FFMA rate for many pairs, by the tiles' way into shared memory for few.
#include "tree_attention.cuh"

namespace {

constexpr int NT = 256, BN = TLC_PAGE;
constexpr float LOG2E = 1.4426950408889634f;

__host__ __device__ constexpr int padded(int hd) { return ((hd + 3) / 4) % 2 ? (hd + 3) / 4 * 4 : (hd + 3) / 4 * 4 + 4; }   // 16-byte rows, an odd number of pieces
__host__ __device__ constexpr int smem_floats(int hd, int rows) { return (rows + BN) * padded(hd) + BN * ((hd + 63) / 64 * 64) + rows * (BN + 4); }

// RM rows of pairs a thread (16 RM a tile), NJ times 64 columns of values.
template <typename T, int RM, int NJ>
__global__ void __launch_bounds__(NT)
tree_attention_kernel(TreeArgs a) {
  asm volatile("griddepcontrol.launch_dependents;");
  tlc_wait(a.q, a.k_new, a.v_new, a.k_pages, a.v_pages, a.block_table, a.slots, a.start, a.cu, a.positions, a.mask, a.out, a.part_o, a.part_ml,
           a.splits);
  constexpr int ROWS = 16 * RM;
  extern __shared__ float4 tree_raw[];
  const int hd = a.hd, hp = padded(hd), hv = NJ * 64, G = a.H / a.KV;
  float* const Q = reinterpret_cast<float*>(tree_raw);
  float* const K = Q + ROWS * hp;
  float* const V = K + BN * hp;
  float* const P = V + BN * hv;                            // [ROWS][BN + 4]
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const T* const q = reinterpret_cast<const T*>(a.q);
  const TreeTake take = tree_plan<NT>(a, blockIdx.x, reinterpret_cast<int*>(tree_raw));
  int b = take.b, unit = take.unit, todo = take.todo;
  TreeSeq s = take.s;
  const float scale2 = a.scale * LOG2E;
  for (bool first_segment = true; todo > 0; first_segment = false) {
    while (unit >= s.units) { unit -= s.units; s = tree_seq(a, ++b); }
    const int item = unit / s.key_tiles, kt0 = unit % s.key_tiles;
    const int g = item / s.row_tiles, r0 = item % s.row_tiles * a.tile_rows;
    const int kt1 = min(s.key_tiles, kt0 + todo);
    const int pairs = min(a.tile_rows, s.n * G - r0);
    const int* const table = a.block_table + (size_t)(s.context_tiles > 0 ? a.slots[b] : 0) * a.max_pages;
    __syncthreads();                                        // the segment before has used its queries
    // the tile's queries
    for (int e = tid; e < ROWS * hp; e += NT) {
      const int r = e / hp, d = e % hp;
      float v = 0.f;
      if (r < pairs && d < hd) {
        const int i = (r0 + r) / G, h = g * G + (r0 + r) % G;
        v = to_f32(q[(size_t)(s.t0 + i) * a.ld_q + (size_t)h * hd + d]);
      }
      Q[e] = v;
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
      __syncthreads();                                      // the tile before has been used
      for (int e = tid; e < BN * hp; e += NT) {
        const int r = e / hp, d = e % hp;
        K[e] = there && r < keys && d < hd ? to_f32(kr[r * ldk + d]) : 0.f;
      }
      bool odd = false;                                     // a value that is no number must not reach rows that do not see it
      for (int e = tid; e < BN * hv; e += NT) {
        const int r = e / hv, d = e % hv;
        const float v = there && r < keys && d < hd ? to_f32(vr[r * ldv + d]) : 0.f;
        V[e] = v;
        odd |= !isfinite(v);
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
    const size_t part = ((size_t)blockIdx.x * 2 + (first_segment ? 0 : 1)) * a.part_rows;
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
        if (tx == 0) { a.part_ml[(part + r) * 2] = m[u]; a.part_ml[(part + r) * 2 + 1] = l[u]; }
#pragma unroll
        for (int c = 0; c < 4 * NJ; c++) {
          const int d = 64 * (c / 4) + tx * 4 + c % 4;
          if (d < hd) a.part_o[(part + r) * hd + d] = o[u][c];
        }
      }
    }
    todo -= kt1 - kt0;
    unit += kt1 - kt0;
  }
}

// Items that several blocks share: o = sum_z o_z 2^(m_z - m) / (sum_z l_z 2^(m_z - m) [+ 2^(sink - m)]).  Every block reads which items those
// are (an entry of splits for each block of the kernel before) and takes its share of their rows: a row a block, the segments shared out
// over the warps, where there are few rows in many segments, else four rows a warp.  Bound by trips to the L2, of which rows take two (the
// statistics, then twelve segments' values at a time); a launch with nothing to add up is over after one.
constexpr int MG_T = 256, MG_WARPS = MG_T / 32, MG_MOST = 512;           // MG_MOST: blocks of the kernel before, at most
constexpr int MG_ROWS = 4;                                               // of a warp
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(MG_T)
tree_merge_kernel(TreeArgs a) {
  tlc_pdl(a.part_o, a.part_ml, a.splits, a.out);
  __shared__ int s_before[MG_MOST], s_warp[MG_WARPS], s_most;
  __shared__ TreeSplit s_split[MG_MOST];
  __shared__ float s_w[MG_MOST], s_red[2 * MG_WARPS], s_acc[MG_WARPS][NV * 32 * VEC];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = a.H / a.KV, hd = a.hd;
  // the items' rows, in fours
  constexpr int EACH = MG_MOST / MG_T;
  int total = 0;
  if (tid == 0) s_most = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const int c = i * MG_T + tid;
    if (i * MG_T >= a.blocks) {
      s_before[c] = 0x7fffffff;
      continue;
    }
    TreeSplit sp = {};
    if (c < a.blocks) sp = a.splits[c];
    s_split[c] = sp;
    const int n = sp.n > 1 ? (sp.pairs + MG_ROWS - 1) / MG_ROWS * MG_ROWS : 0;
    if (sp.n > 1) atomicMax(&s_most, sp.n);
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (i > 0) __syncthreads();
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int before = total + x - n;
#pragma unroll
    for (int w = 0; w < MG_WARPS; w++) {
      if (w < warp) before += s_warp[w];
      total += s_warp[w];
    }
    s_before[c] = before;
  }
  __syncthreads();
  // rounds of some three trips for a row a block; of one, and one for every three segments, for four rows a warp
  const int grid = gridDim.x, wide = grid * MG_WARPS * MG_ROWS;
  const bool together = (total + grid - 1) / grid * 3 < (total + wide - 1) / wide * (1 + (s_most + 2) / 3) || total <= grid;
  for (int at = together ? blockIdx.x : (blockIdx.x * MG_WARPS + warp) * MG_ROWS; at < total; at += together ? grid : wide) {
    int c = 0;                                             // the last block whose rows start at or before this one
#pragma unroll
    for (int step = MG_MOST / 2; step > 0; step >>= 1)
      if (s_before[c + step] <= at) c += step;
    const TreeSplit& item = s_split[c];
    const int c0 = item.c0, n = item.n, r = at - s_before[c];
    auto part = [&](int z, int row) { return ((size_t)(c0 + z) * 2 + (z == 0 ? item.slot0 : 0)) * a.part_rows + row; };
    auto sink_of = [&](int row) { return a.sink && a.sink_values ? a.sink_values[item.g * G + (item.r0 + row) % G] * LOG2E : 0.f; };
    auto place = [&](int row) {
      return reinterpret_cast<T*>(a.out) + (size_t)(item.t0 + (item.r0 + row) / G) * a.out_ld + (size_t)(item.g * G + (item.r0 + row) % G) * hd;
    };
    auto stats = [&](int z, int row) { return z < n && row < item.pairs ? *reinterpret_cast<const float2*>(a.part_ml + part(z, row) * 2) : make_float2(-INFINITY, 0.f); };
    auto values = [&](int z, int row, float (&v)[NV][VEC]) {
      const float* const p = a.part_o + part(z, row) * hd;
#pragma unroll
      for (int e = 0; e < NV; e++) {
        const int d = (lane + 32 * e) * VEC;
        if constexpr (VEC == 4) {
          const float4 f = d < hd ? *reinterpret_cast<const float4*>(p + d) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[e][0] = f.x; v[e][1] = f.y; v[e][2] = f.z; v[e][3] = f.w;
        } else v[e][0] = d < hd ? p[d] : 0.f;
      }
    };
    if (together) {
      if (r >= item.pairs) continue;                       // (filled up to four)
      __syncthreads();                                     // the row before has been read
      const float sv = sink_of(r);
      float m = -INFINITY, l = 0.f, acc[NV][VEC];
#pragma unroll
      for (int e = 0; e < NV; e++)
#pragma unroll
        for (int q = 0; q < VEC; q++) acc[e][q] = 0.f;
      float2 ml[EACH];
#pragma unroll
      for (int i = 0; i < EACH; i++) {
        ml[i] = stats(i * MG_T + tid, r);
        if (ml[i].y != 0.f) m = fmaxf(m, ml[i].x);
      }
      m = warp_max(m);
      if (lane == 0) s_red[warp] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < MG_WARPS; w++) m = fmaxf(m, s_red[w]);
      if (a.sink) m = fmaxf(m, sv);
#pragma unroll
      for (int i = 0; i < EACH; i++)
        if (i * MG_T + tid < n) {
          const float w = ml[i].y != 0.f ? exp2f(ml[i].x - m) : 0.f;
          s_w[i * MG_T + tid] = w;
          if (ml[i].y != 0.f) l += ml[i].y * w;
        }
      l = warp_sum(l);
      if (lane == 0) s_red[MG_WARPS + warp] = l;
      __syncthreads();
      l = 0.f;
#pragma unroll
      for (int w = 0; w < MG_WARPS; w++) l += s_red[MG_WARPS + w];
      constexpr int Z = NV == 1 ? 12 : 4;                  // segments on their way at a time
      for (int z0 = warp; z0 < n; z0 += Z * MG_WARPS) {
        float v[Z][NV][VEC];
#pragma unroll
        for (int z = 0; z < Z; z++)
          if (z0 + z * MG_WARPS < n) values(z0 + z * MG_WARPS, r, v[z]);
#pragma unroll
        for (int z = 0; z < Z; z++) {
          const float w = z0 + z * MG_WARPS < n ? s_w[z0 + z * MG_WARPS] : 0.f;
          if (w == 0.f) continue;
#pragma unroll
          for (int e = 0; e < NV; e++)
#pragma unroll
            for (int q = 0; q < VEC; q++) acc[e][q] = fmaf(v[z][e][q], w, acc[e][q]);
        }
      }
#pragma unroll
      for (int e = 0; e < NV; e++)
#pragma unroll
        for (int q = 0; q < VEC; q++) s_acc[warp][(lane + 32 * e) * VEC + q] = acc[e][q];
      __syncthreads();
      if (tid < hd) {
        const float inv = l == 0.f ? 0.f : 1.0f / (a.sink ? l + exp2f(sv - m) : l);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < MG_WARPS; w++) sum += s_acc[w][tid];
        place(r)[tid] = from_f32<T>(l == 0.f ? 0.f : sum * inv);
      }
      continue;
    }
    // four rows a warp, eight lanes a row for its segments' weights
    constexpr int LANES = 32 / MG_ROWS;
    const int own = r + lane / LANES;
    const float sv = own < item.pairs ? sink_of(own) : 0.f;
    float2 ml = stats(lane % LANES, own);
    float m = ml.y != 0.f ? ml.x : -INFINITY, l = 0.f, acc[MG_ROWS][NV][VEC];
    for (int z = LANES + lane % LANES; z < n; z += LANES) {
      const float2 o = stats(z, own);
      if (o.y != 0.f) m = fmaxf(m, o.x);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (a.sink) m = fmaxf(m, sv);
#pragma unroll
    for (int x = 0; x < MG_ROWS; x++)
#pragma unroll
      for (int e = 0; e < NV; e++)
#pragma unroll
        for (int q = 0; q < VEC; q++) acc[x][e][q] = 0.f;
    for (int base = 0; base < n; base += LANES) {
      if (base > 0) ml = stats(base + lane % LANES, own);
      const float w = ml.y != 0.f ? exp2f(ml.x - m) : 0.f;
      if (ml.y != 0.f) l += ml.y * w;
      constexpr int Z = NV == 1 ? 3 : 1;                   // segments of the four rows on their way at a time
      const int stop = min(n, base + LANES);
      for (int z0 = base; z0 < stop; z0 += Z) {
        float v[Z][MG_ROWS][NV][VEC];
#pragma unroll
        for (int z = 0; z < Z; z++)
#pragma unroll
          for (int x = 0; x < MG_ROWS; x++)
            if (z0 + z < stop && r + x < item.pairs) values(z0 + z, r + x, v[z][x]);
#pragma unroll
        for (int z = 0; z < Z; z++)
#pragma unroll
          for (int x = 0; x < MG_ROWS; x++) {
            const float wz = __shfl_sync(0xffffffffu, w, x * LANES + (z0 + z) % LANES);
            if (z0 + z >= stop || wz == 0.f || r + x >= item.pairs) continue;
#pragma unroll
            for (int e = 0; e < NV; e++)
#pragma unroll
              for (int q = 0; q < VEC; q++) acc[x][e][q] = fmaf(v[z][x][e][q], wz, acc[x][e][q]);
          }
      }
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const float inv = l == 0.f ? 0.f : 1.0f / (a.sink ? l + exp2f(sv - m) : l);
#pragma unroll
    for (int x = 0; x < MG_ROWS; x++) {
      const float f = __shfl_sync(0xffffffffu, inv, x * LANES);
      const bool none = __shfl_sync(0xffffffffu, l, x * LANES) == 0.f;
      if (r + x >= item.pairs) continue;
      T* const to = place(r + x);
#pragma unroll
      for (int e = 0; e < NV; e++)
#pragma unroll
        for (int q = 0; q < VEC; q++) {
          const int d = (lane + 32 * e) * VEC + q;
          if (d < hd) to[d] = from_f32<T>(none ? 0.f : acc[x][e][q] * f);
        }
    }
  }
}

template <typename T> void run_merge(const TreeArgs& a, cudaStream_t stream) {
  auto* const k = a.hd % 4 != 0 ? tree_merge_kernel<T, 1, 8> : a.hd <= 128 ? tree_merge_kernel<T, 4, 1> : tree_merge_kernel<T, 4, 2>;
  const long long rows = (long long)a.T * a.H, most = 148 * 4;           // a block a row at most, four to an SM
  tlc_launch(k, dim3((unsigned)(rows < most ? rows : most)), dim3(MG_T), 0, stream, a);
}

template <typename T, int RM> int run_simt(const TreeArgs& a, cudaStream_t stream) {
  const int nj = (a.hd + 63) / 64, smem = smem_floats(a.hd, 16 * RM) * (int)sizeof(float);
  auto* const k = nj == 1 ? tree_attention_kernel<T, RM, 1> : nj == 2 ? tree_attention_kernel<T, RM, 2> : tree_attention_kernel<T, RM, 4>;
  const int full = nj <= 2 ? smem : smem + BN * (256 - nj * 64) * (int)sizeof(float);
  if (full > 48 * 1024 && cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, full) != cudaSuccess)
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
  static int sms = 0;
  if (sms == 0) { int dev = 0; cudaGetDevice(&dev); cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev); }
  Cut c;
  const int G = H / KV;
  c.tc = tlc_tree_attention_tc_takes(dtype, aligned, H, KV, hd, n_pages);
  c.rows = c.tc ? 256 : (long long)max_new * G > 16 ? 64 : 16;
  c.tile_rows = c.tc ? 128 / G * G * 2 : c.rows;
  const long long kt = ((long long)max_context + BN - 1) / BN + (max_new + BN - 1) / BN;
  c.units = (((long long)T * G + c.tile_rows - 1) / c.tile_rows + B) * KV * kt;
  const long long wave = (long long)sms * (c.tc ? 1 : 2);
  c.blocks = (int)(c.units < wave ? (c.units < 1 ? 1 : c.units) : wave);
  if (c.blocks > MG_MOST) c.blocks = MG_MOST;
  c.scratch = (long long)c.blocks * (2 * c.rows * (hd + 2) * 4 + (long long)sizeof(TreeSplit));
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
  TLC_REQUIRE(c.units < (1ll << 31), "tree_attention: %d rows over %d keys are too many", T, max_context);
  TreeArgs a = {};
  a.q = q; a.k_new = k_new; a.v_new = v_new; a.k_pages = k_pages; a.v_pages = v_pages;
  a.ld_q = ld_q; a.ld_k = ld_k; a.ld_v = ld_v; a.n_pages = n_pages;
  a.block_table = block_table; a.slots = slots; a.start = start; a.cu = cu_seqlens; a.positions = positions; a.mask = mask;
  a.n_slots = n_slots; a.max_pages = max_pages; a.words = words;
  a.out = out; a.out_ld = out_ld; a.B = B; a.T = T; a.H = H; a.KV = KV; a.hd = hd;
  a.scale = scale; a.window = window > 0 ? window : 0; a.softcap = softcap; a.sink = sink; a.sink_values = sink_values;
  a.max_context = max_context;
  a.tile_rows = c.tile_rows;
  a.blocks = c.blocks;
  a.part_rows = c.rows;
  a.part_o = (float*)scratch;
  a.part_ml = a.part_o + (size_t)c.blocks * 2 * c.rows * hd;
  a.splits = (TreeSplit*)(a.part_ml + (size_t)c.blocks * 2 * c.rows * 2);
  if (const int rc = c.tc ? tlc_tree_attention_tc(a, stream) : tlc_tree_attention_simt(a, dtype, c.rows, stream)) return rc;
  TLC_DISPATCH_DTYPE(dtype, E, run_merge<E>(a, stream));
  TLC_CHECK_LAUNCH("tree_attention(merge)");
  return 0;
}
