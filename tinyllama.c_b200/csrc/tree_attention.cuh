// What the kernels of tree attention share: the arguments, which work a block takes, and where its partial results go.
#pragma once
#include "common.cuh"

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
  int max_context;
  int tile_rows;                                          // (row, head of the group) pairs of a tile
  int blocks;
  float *part_o, *part_ml;                                // [blocks, 2, most rows of a tile, hd] and the same with 2 for hd
  int part_rows;                                          // most rows of a tile
  int* plan;                                              // [B + 1] units before each request, [B] key tiles of each
};

// A request: its rows, how much of its context there is to see, and in how many units of work (one key/value head, one tile of
// rows, one tile of 64 keys) it comes.
struct TreeSeq {
  int t0, n, context, first_tile, context_tiles, key_tiles, row_tiles, units;
};

__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int b) {
  TreeSeq s;
  s.t0 = min(max(a.cu[b], 0), a.T);
  s.n = min(max(a.cu[b + 1], s.t0), a.T) - s.t0;
  const int slot = a.slots[b];
  s.context = slot >= 0 && slot < a.n_slots ? min(max(a.start[b], 0), min(a.max_context, (int)min((long long)a.max_pages * TLC_PAGE, 2147483647ll))) : 0;
  s.first_tile = a.window > 0 ? max(0, s.context + 1 - a.window) / TLC_PAGE : 0;
  s.context_tiles = (s.context + TLC_PAGE - 1) / TLC_PAGE - s.first_tile;
  s.key_tiles = s.context_tiles + (s.n + TLC_PAGE - 1) / TLC_PAGE;
  s.row_tiles = (s.n * (a.H / a.KV) + a.tile_rows - 1) / a.tile_rows;
  s.units = a.KV * s.row_tiles * s.key_tiles;
  return s;
}

// Units are numbered request by request, within it key/value head by head, tile by tile of rows, and tile by tile of keys; block c of n takes
// [c W / n, (c + 1) W / n) of all W (n at most W): every block the same work, however unequal the requests are, and the tiles of keys of one (request, head, row
// tile) - an item - lie in consecutive blocks.  What a block has of an item is a segment.  The item that a block begins with may have
// started in an earlier block and the one it ends with may go on in a later one: these segments' sums are left in part_o (slot 0 for the first
// segment, 1 for the last), and another kernel adds them up.
__device__ __forceinline__ int tree_blocks(long long W, int n) { return (int)(W < n ? W : n); }      // fewer units than blocks: one each, and the rest none
__device__ __forceinline__ long long tree_first(long long W, int c, int n) { return c * W / n; }
__device__ __forceinline__ int tree_block_of(long long W, long long u, int n) { return (int)(((u + 1) * n - 1) / W); }

// All threads of a block of NT call it: which request the first unit of block c is in, and which of that request's it is.
// count: how many units the block takes.  Block 0 leaves the plan that the merging kernel reads.
template <int NT> __device__ __forceinline__ void tree_plan(const TreeArgs& a, int c, int* at_seq, int* at_unit, long long* count) {
  __shared__ long long red[NT / 32 + 1];
  __shared__ int s_seq, s_unit;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int each = (a.B + NT - 1) / NT, b0 = min(a.B, tid * each), b1 = min(a.B, b0 + each);
  long long mine = 0;
  for (int b = b0; b < b1; b++) mine += tree_seq(a, b).units;
  long long x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (tid == 0) s_seq = -1;
  if (lane == 31) red[warp] = x;
  __syncthreads();
  long long before = x - mine, W = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; w++) {
    if (w < warp) before += red[w];
    W += red[w];
  }
  const int n = tree_blocks(W, a.blocks);
  const long long first = c < n ? tree_first(W, c, n) : -1;
  for (int b = b0; b < b1; b++) {
    const TreeSeq s = tree_seq(a, b);
    if (first >= before && first < before + s.units) { s_seq = b; s_unit = (int)(first - before); }
    if (c == 0) { a.plan[b] = (int)before; a.plan[a.B + 1 + b] = s.key_tiles; }
    before += s.units;
  }
  if (c == 0 && tid == 0) a.plan[a.B] = (int)W;
  __syncthreads();
  *at_seq = s_seq;
  *at_unit = s_unit;
  *count = c < n ? tree_first(W, c + 1, n) - first : 0;
}

// Whether the draft's row i (position pos) sees draft j (position pos_j).
__device__ __forceinline__ bool tree_sees(const TreeArgs& a, int t0, int i, int j) {
  if (a.mask) {
    if ((j >> 5) >= a.words || !((unsigned)a.mask[(size_t)(t0 + i) * a.words + (j >> 5)] >> (j & 31) & 1)) return false;
  } else if (j > i) return false;
  return a.window <= 0 || a.positions[t0 + j] > a.positions[t0 + i] - a.window;
}

int tlc_tree_attention_simt(const TreeArgs& a, int dtype, int rows, cudaStream_t stream);
int tlc_tree_attention_tc(const TreeArgs& a, cudaStream_t stream);
bool tlc_tree_attention_tc_takes(int dtype, int aligned, int H, int KV, int hd, long long n_pages);
