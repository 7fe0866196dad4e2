// What the kernels of tree attention share: the arguments, which work a block takes, and where its partial results go.
#pragma once
#include "common.cuh"
#include "mbarrier.cuh"

// What block c leaves for the kernel that adds up partial results: an item whose segments are those of blocks c0 .. c0 + n - 1 (n 0: none).
struct TreeSplit {
  int n, c0, slot0;                                       // slot0: where block c0's is (the others' are in slot 0)
  int t0, r0, pairs, g;                                   // the request's first row, the item's first pair of it, how many, the key/value head
  int pad;
};

struct TreeArgs {
  const void *q, *k_new, *v_new, *k_pages, *v_pages;      // [T, H * hd], [T, KV * hd] twice, [n_pages, KV, 64, hd] twice
  int ld_q, ld_k, ld_v, n_pages;                          // row strides in elements
  const int *block_table, *slots, *start, *cu, *positions, *mask;      // mask [T, words] or NULL: every row sees the drafts up to itself
  int n_slots, max_pages, words;
  void* out;
  int out_ld, B, T, H, KV, hd;
  float scale;
  int window;
  float softcap;
  int sink;
  const float* sink_values;
  int max_context, max_new;                               // a longer context is cut, and so is a request of more rows (TREE_MORE_ROWS is reported)
  int G;                                                  // query heads of a key/value head
  int vec, vec_out;                                       // every input row, every output row starts on a boundary of four elements, with heads of fours
  int tile_rows;                                          // (row, head of the group) pairs of a tile
  int blocks;
  float *part_o, *part_ml;                                // [blocks, 2, hd in fours, most rows of a tile, 4] and [blocks, 2, most rows of a tile, 2]
  int part_rows;                                          // most rows of a tile
  struct TreeSplit* splits;                               // [blocks]
  ErrWords* err;                                          // or NULL
};

constexpr int TREE_MORE_ROWS = 60;                        // code of the error word

// a / b of numbers that are not negative: by a 32-bit reciprocal where they are small (a plan is a chain of divisions, an integer one
// takes four times as long)
__device__ __forceinline__ int tree_div(int a, int b) {
  if (a >= 1 << 22) return a / b;
  int q = (int)__fdividef((float)a, (float)b);            // off by one at most
  const int r = a - q * b;
  return q + (r >= b ? 1 : 0) - (r < 0 ? 1 : 0);
}

// A request: its rows, how much of its context there is to see, and in how many units of work (one key/value head, one tile of
// rows, one tile of 64 keys) it comes.
struct TreeSeq {
  int t0, n, context, first_tile, context_tiles, key_tiles, row_tiles, units;
};

__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int b) {
  TreeSeq s;
  s.t0 = min(max(a.cu[b], 0), a.T);
  s.n = min(min(max(a.cu[b + 1], s.t0), a.T) - s.t0, a.max_new);
  const int slot = a.slots[b];
  s.context = slot >= 0 && slot < a.n_slots ? min(max(a.start[b], 0), min(a.max_context, (int)min((long long)a.max_pages * TLC_PAGE, 2147483647ll))) : 0;
  s.first_tile = a.window > 0 ? max(0, s.context - (a.window - 1)) / TLC_PAGE : 0;
  s.context_tiles = (int)(((unsigned)s.context + (TLC_PAGE - 1)) / TLC_PAGE) - s.first_tile;     // (of a context up to 2^31 - 1)
  s.key_tiles = s.context_tiles + (s.n + TLC_PAGE - 1) / TLC_PAGE;
  s.row_tiles = tree_div(s.n * a.G + a.tile_rows - 1, a.tile_rows);
  s.units = a.KV * s.row_tiles * s.key_tiles;
  return s;
}

// Units are numbered request by request, within it key/value head by head, tile by tile of rows, and tile by tile of keys; the tiles of keys of one
// (request, head, row tile) are an item, what a block has of an item is a segment.  Segments whose item other blocks share leave their sums in
// part_o, and another kernel adds them up.  Two ways to give the n blocks their work:
//   * items in equal pieces of at most P units, a piece a block, with the smallest P for which the pieces are at most n;
//   * where that P is more than SLACK above the mean W / n (many items, of unequal lengths): block c takes the next W / n units, whatever
//     they belong to; the item that it begins with may have started in an earlier block and the one it ends with may go on in a
//     later one (part_o has a slot for each).
// A second segment costs a block about what SLACK units do (its queries, the products' way in, its sums: 16 requests of 150 to 6,000 keys in
// pieces 35 us, in equal shares 50).
constexpr int TREE_SLACK = 4, TREE_MOST_SEQS = 2048;      // requests whose pieces are looked at

struct TreeShare {
  int n, per, more;
  __device__ __forceinline__ TreeShare(int W, int blocks) : n(min(W, blocks)), per(n > 0 ? tree_div(W, n) : 0), more(W - per * n) {}
  __device__ __forceinline__ int first(int c) const { return c * per + min(c, more); }
  __device__ __forceinline__ int block_of(int u) const { return u < more * (per + 1) ? tree_div(u, per + 1) : more + tree_div(u - more * (per + 1), per); }
};

struct TreeTake {
  int b, item, tile, todo;                                // the block begins with key tile `tile` of item `item` of request b and takes `todo` units
  TreeSeq s;                                              // request b
};

template <int NT> __device__ __forceinline__ int tree_before(int mine, int* red) {     // the sum over the threads before; red: NT / 32 ints
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) red[warp] = x;
  __syncthreads();
  int before = x - mine;
#pragma unroll
  for (int w = 0; w < NT / 32; w++)
    if (w < warp) before += red[w];
  return before;
}

// All threads of a block of NT call it.  room: 2 * min(B, TREE_MOST_SEQS) ints of shared memory.  Leaves block c's entry of splits.
template <int NT> __device__ __forceinline__ TreeTake tree_plan(const TreeArgs& a, int c, int* room) {
  __shared__ int red_w[NT / 32], red_i[NT / 32], red_b[NT / 32], s_piece[TREE_SLACK + 1];
  __shared__ TreeTake s_take;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int each = (a.B + NT - 1) / NT, b0 = min(a.B, tid * each), b1 = min(a.B, b0 + each);
  const bool look = a.B <= TREE_MOST_SEQS;
  TreeSeq s = {};
  int units = 0, items = 0;
  for (int b = b0; b < b1; b++) {
    s = tree_seq(a, b);
    units += s.units;
    items += a.KV * s.row_tiles;
    if (c == 0 && a.err && min(a.cu[b + 1], a.T) - s.t0 > a.max_new) {
      atomicExch(&a.err->flag, TREE_MORE_ROWS);
      *(volatile int*)a.err->host = TREE_MORE_ROWS;
    }
    if (look) { room[2 * b] = a.KV * s.row_tiles; room[2 * b + 1] = s.key_tiles; }
  }
  const int w_sum = __reduce_add_sync(0xffffffffu, units), i_sum = __reduce_add_sync(0xffffffffu, items);
  if (lane == 0) { red_w[warp] = w_sum; red_i[warp] = i_sum; }
  if (tid == 0) s_take.todo = 0;
  __syncthreads();
  int W = 0, I = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; w++) { W += red_w[w]; I += red_i[w]; }
  const TreeShare share(W, a.blocks);
  // the smallest P of mean .. mean + SLACK for which there are blocks enough, a warp each
  static_assert(NT / 32 > TREE_SLACK, "a warp for every candidate");
  if (warp <= TREE_SLACK) {
    int n = 0x7fffffff;
    const int p = tree_div(W + a.blocks - 1, a.blocks) + warp;
    if (look && I <= a.blocks && W > 0) {
      n = 0;
      for (int b = lane; b < a.B; b += 32) n += room[2 * b] * tree_div(room[2 * b + 1] + p - 1, p);
      n = (int)__reduce_add_sync(0xffffffffu, n);
    }
    if (lane == 0) s_piece[warp] = n <= a.blocks ? p : 0;
  }
  __syncthreads();
  int piece = 0;
#pragma unroll
  for (int w = TREE_SLACK; w >= 0; w--) piece = s_piece[w] > 0 ? s_piece[w] : piece;
  TreeSplit split = {};
  if (piece > 0) {
    int mine = 0;
    for (int b = b0; b < b1; b++) mine += room[2 * b] * tree_div(room[2 * b + 1] + piece - 1, piece);
    int before = tree_before<NT>(mine, red_b);
    for (int b = b0; b < b1; b++) {
      const int n = tree_div(room[2 * b + 1] + piece - 1, piece), here = room[2 * b] * n;
      if (c >= before && c < before + here) {
        if (each > 1) s = tree_seq(a, b);
        const int item = tree_div(c - before, n), k = c - before - item * n;
        // (n is at most 512: the products of more tiles may pass 32 bits)
        const bool small = s.key_tiles < 1 << 22;
        const int whole = small ? 0 : s.key_tiles / n, rest = s.key_tiles - whole * n;
        const int lo = k * whole + tree_div(k * rest, n);
        s_take = TreeTake{b, item, lo, (k + 1) * whole + tree_div((k + 1) * rest, n) - lo, s};
        if (k == 0 && n > 1) {
          const int g = tree_div(item, s.row_tiles), r0 = (item - g * s.row_tiles) * a.tile_rows;
          split = TreeSplit{n, c, 0, s.t0, r0, min(a.tile_rows, s.n * a.G - r0), g, 0};
        }
        a.splits[c] = split;
      }
      before += here;
    }
  } else {
    int before = tree_before<NT>(units, red_b);
    const int first = c < share.n ? share.first(c) : -1;
    for (int b = b0; b < b1; b++) {
      if (each > 1) s = tree_seq(a, b);
      if (first >= before && first < before + s.units) {
        const int unit = first - before, item = tree_div(unit, s.key_tiles), tile = unit - item * s.key_tiles, u0 = first - tile;
        s_take = TreeTake{b, item, tile, share.first(c + 1) - first, s};
        if (tile > 0 && share.block_of(u0) == c - 1) {
          const int g = tree_div(item, s.row_tiles), r0 = (item - g * s.row_tiles) * a.tile_rows;
          split = TreeSplit{share.block_of(u0 + s.key_tiles - 1) - c + 2, c - 1, share.first(c - 1) < u0 ? 1 : 0, s.t0, r0,
                            min(a.tile_rows, s.n * a.G - r0), g, 0};
        }
        a.splits[c] = split;
      }
      before += s.units;
    }
  }
  __syncthreads();
  const TreeTake take = s_take;
  if (take.todo == 0 && tid == 0) a.splits[c] = TreeSplit{};             // nothing to do
  return take;
}

// Whether the draft's row i (position pos) sees draft j (position pos_j).
__device__ __forceinline__ bool tree_sees(const TreeArgs& a, int t0, int i, int j) {
  if (a.mask) {
    if ((j >> 5) >= a.words || !((unsigned)a.mask[(size_t)(t0 + i) * a.words + (j >> 5)] >> (j & 31) & 1)) return false;
  } else if (j > i) return false;
  return a.window <= 0 || a.positions[t0 + j] > a.positions[t0 + i] - a.window;
}

// The four values from column 4 c on of row r in block z's slot: lanes that have a row each write whole lines, and readers take four rows.
__device__ __forceinline__ float4* tree_part(const TreeArgs& a, int z, int slot, int c, int r) {
  return reinterpret_cast<float4*>(a.part_o) + (((size_t)z * 2 + slot) * ((a.hd + 3) / 4) + c) * a.part_rows + r;
}
__device__ __forceinline__ float2* tree_part_ml(const TreeArgs& a, int z, int slot, int r) {
  return reinterpret_cast<float2*>(a.part_ml) + ((size_t)z * 2 + slot) * a.part_rows + r;
}

int tlc_tree_attention_simt(const TreeArgs& a, int dtype, int rows, cudaStream_t stream);
int tlc_tree_attention_tc(const TreeArgs& a, cudaStream_t stream);
bool tlc_tree_attention_tc_takes(int dtype, int aligned, int H, int KV, int hd, long long n_pages);
