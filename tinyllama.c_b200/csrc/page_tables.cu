// Pages of the key/value store handed out and taken back on the GPU, what a step's rows are told about their places, and
// rows stored at places.
//
// CodeClaper/tinyllama.c keeps a free list of token slots on the host and maps a request's positions to them one by one
// (kvcache.c:70-120).  Here the pool is three arrays in device memory: refs [n_pages] counts the block table's entries that
// name a page (0: the page is free; more than 1: beams share it), lengths [n_slots] says how many positions a slot holds, and
// row s of block_table names the pages of slot s, its first ceil(lengths[s] / 64) entries.  A step that only the GPU knows
// (how many drafted tokens were accepted, which beams go on) then needs no trip to the host.
//
// None of these kernels lets its successor start early (no griddepcontrol.launch_dependents): kernels of a step may fetch
// block-table rows and cache contents ahead of their own wait.
#include "common.cuh"

namespace {

constexpr int RT = 1024;                 // threads of the resizing block
constexpr int MAX_REQUESTS = 4096;       // of one call: their sums and pages lie in shared memory
constexpr int PER = 16;                  // entries of refs a thread looks at a time (four 16-byte loads)

// codes of the status word (the largest that occurred stays until the caller clears it)
enum { ST_FULL = 1, ST_LENGTH = 2, ST_SLOT = 3, ST_TABLE = 4, ST_SHARED = 5 };

__device__ __forceinline__ int pages_of(int n) { return (int)(((unsigned)n + (TLC_PAGE - 1)) / TLC_PAGE); }

// exclusive prefix sum of v over the block; total: the block's sum.  red: 33 values of shared memory.
template <typename V> __device__ __forceinline__ V block_prefix(V v, V* red, V* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  V x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = x;
  __syncthreads();
  if (warp == 0) {
    const V w = lane < nw ? red[lane] : V(0);
    V s = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const V y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    red[lane] = s - w;
    if (lane == 31) red[32] = s;
  }
  __syncthreads();
  *total = red[32];
  return red[warp] + x - v;
}

// the last i of 0..n-1 with sum[i] <= at (sum ascending, sum[0] <= at); entries of equal sums: the last, which is the one that has any
__device__ __forceinline__ int find_sum(const int* sum, int n, int at) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sum[mid] <= at) lo = mid; else hi = mid;
  }
  return lo;
}

// One block does all of it: which page is the p-th lowest free one depends on every page before it, and what a step takes is
// few pages of a pool that is looked through from the start.  Bound by trips to the L2: the requests, their lengths, the last pages'
// counts, then a round for every 16,384 pages looked at (the first round's counts are fetched at the start); in a round the free pages go
// into a list, and the list into the table, a page a thread (700 requests that take 800 pages: 22 us where a thread placed all the pages
// it had found, one after the other; now 9 us, 10 where they give them back, and 4 to 5 us for 8 requests).  Everything another thread of the block may have changed is read past the L1 (__ldcg).
struct Request { int slot, have, need; };             // slot -1: nothing to do

__global__ void __launch_bounds__(RT)
page_resize_kernel(int* block_table, int n_slots, int max_pages, int* refs, int n_pages, int* lengths, const int* slots,
                   const int* want, int B, int* status) {
  tlc_wait(block_table, refs, lengths, slots, want, status);
  extern __shared__ int resize_room[];
  int* const list = resize_room;                      // [RT * PER] free pages of a round
  int* const take = list + RT * PER;                  // [B + 1] pages taken by the requests before
  int* const give = take + B + 1;                     // [B + 1] pages given back by them
  Request* const request = reinterpret_cast<Request*>(give + B + 1);
  __shared__ long long red[33];
  __shared__ int s_bad;
  const int tid = threadIdx.x;
  constexpr int LENGTH = 0x7fffffff, MINE = MAX_REQUESTS / RT;      // requests of a thread, one after the other
  if (tid == 0) s_bad = 0;
  auto bad_so_far = [&]() {
    __syncthreads();
    const int c = s_bad;
    __syncthreads();
    return c;
  };
  const bool vec = (reinterpret_cast<uintptr_t>(refs) & 15) == 0;
  auto load = [&](int at, int (&v)[PER]) {
    if (vec && at + PER <= n_pages) {
#pragma unroll
      for (int q = 0; q < PER / 4; q++) {
        const int4 x = __ldcg(reinterpret_cast<const int4*>(refs + at) + q);
        v[4 * q] = x.x; v[4 * q + 1] = x.y; v[4 * q + 2] = x.z; v[4 * q + 3] = x.w;
      }
    } else {
#pragma unroll
      for (int q = 0; q < PER; q++) v[q] = at + q < n_pages ? __ldcg(refs + at + q) : 1;
    }
  };
  int v[PER];
  load(tid * PER, v);                                 // (loaded again where pages are given back)
  // 1. each request's slot is claimed (by the sign of its length); what the request takes or gives back is added up
  const int each = (B + RT - 1) / RT, b0 = min(B, tid * each), b1 = min(B, b0 + each);
  int slot[MINE], last[MINE], old[MINE], t_of[MINE], g_of[MINE], bad = 0;    // slot -1: none, or not claimed here; last: a page that is grown in
  long long mine = 0;                                 // pages taken, and pages given back in the upper half: below 2^31 each, see tlc_page_resize
#pragma unroll
  for (int i = 0; i < MINE; i++) {
    slot[i] = last[i] = -1;
    t_of[i] = g_of[i] = old[i] = 0;
    const int b = b0 + i;
    if (b >= b1) continue;
    const int s = slots[b], w = want[b];
    if (s >= n_slots) bad = max(bad, (int)ST_SLOT);
    if (s < 0 || s >= n_slots) { request[b] = Request{-1, 0, 0}; continue; }
    old[i] = atomicOr(lengths + s, ~LENGTH);
    const int have = pages_of(old[i] & LENGTH), need = pages_of(max(w, 0));
    request[b] = Request{s, have, need};
    if (old[i] < 0) { bad = max(bad, (int)ST_SLOT); continue; }          // named twice (or no length at all)
    slot[i] = s;
    if (w < 0 || need > max_pages || have > max_pages) { bad = max(bad, (int)ST_LENGTH); continue; }
    t_of[i] = max(0, need - have);
    g_of[i] = max(0, have - need);
    if (w > old[i] && old[i] % TLC_PAGE != 0) {
      last[i] = __ldcg(block_table + (size_t)s * max_pages + have - 1);
      if (last[i] < 0 || last[i] >= n_pages) { bad = max(bad, (int)ST_TABLE); last[i] = -1; }
    }
    mine += (long long)t_of[i] | ((long long)g_of[i] << 32);
  }
  long long total;
  const long long before = block_prefix<long long>(mine, red, &total);
  int t_at = (int)(before & 0xffffffff), g_at = (int)(before >> 32);
#pragma unroll
  for (int i = 0; i < MINE; i++) {
    if (b0 + i >= b1) continue;
    take[b0 + i] = t_at;
    give[b0 + i] = g_at;
    t_at += t_of[i];
    g_at += g_of[i];
  }
  const int n_take = (int)(total & 0xffffffff), n_give = (int)(total >> 32);
  if (tid == 0) { take[B] = n_take; give[B] = n_give; }
  if (bad) atomicMax(&s_bad, bad);
  // the table entry of the i-th page given back, and of the i-th page taken
  auto given = [&](int i) {
    const int b = find_sum(give, B + 1, i);
    return block_table + (size_t)request[b].slot * max_pages + request[b].need + i - give[b];
  };
  auto taken = [&](int i) {
    const int b = find_sum(take, B + 1, i);
    return block_table + (size_t)request[b].slot * max_pages + request[b].have + i - take[b];
  };
  if (bad_so_far() == 0) {
    // 2. pages given back: one entry less each that names them
    if (n_give > 0) {
      for (int i = tid; i < n_give; i += RT) {
        const int p = __ldcg(given(i));
        if (p < 0 || p >= n_pages || atomicSub(refs + p, 1) <= 0) atomicMax(&s_bad, (int)ST_TABLE);
      }
      __syncthreads();
      load(tid * PER, v);
    }
    // a slot that grows inside its last page must have that page to itself
#pragma unroll
    for (int i = 0; i < MINE; i++) {
      if (last[i] < 0) continue;
      const int n = __ldcg(refs + last[i]);
      if (n != 1) atomicMax(&s_bad, n < 1 ? (int)ST_TABLE : (int)ST_SHARED);
    }
    int code = bad_so_far();
    // 3. the lowest free pages, request by request
    int found = 0;
    if (code == 0 && n_take > 0) {
      for (int base = 0; base < n_pages && found < n_take; base += RT * PER) {
        const int at = base + tid * PER;
        int n = 0;
        unsigned free = 0;
#pragma unroll
        for (int q = 0; q < PER; q++) {
          n += v[q] == 0;
          free |= (v[q] == 0 ? 1u : 0u) << q;
        }
        load(at + RT * PER, v);                        // the next round's, on their way during this one's sum
        long long all;
        int rank = (int)block_prefix<long long>(n, red, &all);
        const int most = min((int)all, n_take - found);
        for (; free != 0 && rank < most; free &= free - 1, rank++) list[rank] = at + __ffs(free) - 1;
        __syncthreads();
        for (int i = tid; i < most; i += RT) {
          *taken(found + i) = list[i];
          refs[list[i]] = 1;
        }
        found += most;                                 // (the list is written again after the next sum's barriers)
      }
      if (found < n_take) code = ST_FULL;              // (every thread knows)
    }
    __syncthreads();
    // 4. kept, or all of it undone
    if (code == 0) {
      for (int i = tid; i < n_give; i += RT) *given(i) = 0;
    } else {
      for (int i = tid; i < found; i += RT) {
        int* const e = taken(i);
        refs[__ldcg(e)] = 0;
        *e = 0;
      }
      __syncthreads();                                 // (a page given back may have been taken)
      for (int i = tid; i < n_give; i += RT) {
        const int p = __ldcg(given(i));
        if (p >= 0 && p < n_pages) atomicAdd(refs + p, 1);
      }
      if (tid == 0) s_bad = code;
    }
  }
  const int code = bad_so_far();
#pragma unroll
  for (int i = 0; i < MINE; i++)
    if (slot[i] >= 0) lengths[slot[i]] = code == 0 ? want[b0 + i] : old[i];
  if (code != 0 && tid == 0) atomicMax(status, code);
}

// ---- what a step's rows are told -----------------------------------------------------------------------
constexpr int MT = 256;

// Row t of request b (its i-th): sequence b, position start[b] + i, place page * 64 + offset of that position.  With parents a row is
// a drafted token: parent[t] is the draft it follows (by its index among the request's, always a smaller one; -1: the context), its
// depth is the number of drafts above it, its position start[b] + depth, and mask [T, words] has a bit for each of those and itself.
// Such rows have no place unless `keep` accepts them.  With lengths [n_slots] a row has a place only where its slot holds the position: entries behind
// a slot's pages are 0, and page 0 is somebody's.  Every block adds up the requests' rows by itself (a few loads a
// thread), so nothing has to be handed from block to block.  Bound by trips to the L2, three after one another: 3.4 us for 8 rows, 4.3 for
// 53,000 rows of 700 requests.
__global__ void __launch_bounds__(MT)
row_maps_kernel(const int* __restrict__ block_table, int n_slots, int max_pages, const int* __restrict__ slots,
                const int* __restrict__ lengths, const int* __restrict__ start, const int* __restrict__ rows_of, int B, int T,
                const int* __restrict__ parents, const unsigned char* __restrict__ keep, int words, int* __restrict__ cu, int* __restrict__ row_seq,
                int* __restrict__ positions, int* __restrict__ row_map, int* __restrict__ mask) {
  tlc_wait(block_table, slots, lengths, start, rows_of, parents, keep, cu, row_seq, positions, row_map, mask);
  extern __shared__ int sum[];                        // [B + 1]
  __shared__ long long red[33];
  const int tid = threadIdx.x, each = (B + MT - 1) / MT, b0 = min(B, tid * each), b1 = min(B, b0 + each);
  long long mine = 0;
  for (int b = b0; b < b1; b++) mine += max(0, rows_of[b]);
  long long total, at = block_prefix<long long>(mine, red, &total);
  for (int b = b0; b < b1; b++) {
    sum[b] = (int)min((long long)T, at);              // rows for which there is no room are left out
    at += max(0, rows_of[b]);
  }
  if (tid == 0) sum[B] = (int)min((long long)T, total);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int b = tid; b <= B; b += MT) cu[b] = sum[b];
  const int t = blockIdx.x * MT + tid;
  if (t >= T) return;
  int* const bits = mask ? mask + (size_t)t * words : nullptr;
  if (t >= sum[B]) {                                  // behind the last request
    row_seq[t] = -1;
    positions[t] = 0;
    row_map[t] = -1;
    for (int w = 0; w < words; w++) bits[w] = 0;
    return;
  }
  const int b = find_sum(sum, B + 1, t), i = t - sum[b];
  int depth = i;
  bool lost = false;
  if (parents) {
    const int* const up = parents + sum[b];
    depth = 0;
    lost = i >> 5 >= words;                           // (the mask has no bit for it)
    int word = i >> 5, here = i;
    unsigned acc = 1u << (i & 31);
    for (int w = words - 1; w > word; w--) bits[w] = 0;
    while (!lost) {                                   // up the tree: indices fall, so the words are finished from the last to the first
      const int p = up[here];
      if (p == -1) break;
      if (p < 0 || p >= here) { lost = true; break; }
      depth++;
      here = p;
      if (p >> 5 != word) {
        if (word < words) bits[word] = (int)acc;
        for (int w = min(word, words) - 1; w > p >> 5; w--) bits[w] = 0;
        word = p >> 5;
        acc = 0;
      }
      acc |= 1u << (p & 31);
    }
    if (word < words) bits[word] = (int)acc;
    for (int w = min(word, words) - 1; w >= 0; w--) bits[w] = 0;
    if (lost) {                                       // no bit, or no parent that could be: the row sees no draft and is not kept
      for (int w = 0; w < words; w++) bits[w] = 0;
      depth = 0;
    }
  }
  const long long position = (long long)max(0, start[b]) + depth;
  row_seq[t] = b;
  positions[t] = (int)position;
  int place = -1;
  const int s = slots[b];
  if (!lost && (keep ? keep[t] != 0 : parents == nullptr) && s >= 0 && s < n_slots && position < (long long)max_pages * TLC_PAGE) {
    const int p = block_table[(size_t)s * max_pages + position / TLC_PAGE];
    if (p >= 0 && p < (1 << 25) && (!lengths || position < lengths[s])) place = p * TLC_PAGE + (int)(position % TLC_PAGE);
  }
  row_map[t] = place;
}

// ---- rows to their places ----------------------------------------------------------------------------------
// k, v [L, T, KV * hd] (rows of any stride) to pages [L, n_pages, KV, 64, hd]; rows without a place stay out.  A warp takes a row of a layer,
// keys and values together; a lane moves 16 bytes of a page at a time, and both rows' loads are on their way before the first store.
// Bound by HBM: 8,800 rows of 2 x 128 values in two layers from 32 bits are 54 MB in all, 10.0 us (5.4 TB/s).
template <typename S, typename D, int VEC> struct Pack;
template <typename D> struct Pack<D, D, 1> {
  D x;
  __device__ __forceinline__ void load(const D* p) { x = *p; }
  __device__ __forceinline__ void store(D* p) const { *p = x; }
};
template <> struct Pack<float, __nv_bfloat16, 1> {
  __nv_bfloat16 x;
  __device__ __forceinline__ void load(const float* p) { x = __float2bfloat16_rn(*p); }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *p = x; }
};
template <> struct Pack<__nv_bfloat16, float, 1> {
  float x;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { x = __bfloat162float(*p); }
  __device__ __forceinline__ void store(float* p) const { *p = x; }
};
template <typename D> struct Pack<D, D, 16 / sizeof(D)> {
  uint4 x;
  __device__ __forceinline__ void load(const D* p) { x = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void store(D* p) const { *reinterpret_cast<uint4*>(p) = x; }
};
template <> struct Pack<float, __nv_bfloat16, 8> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = __ldcs(reinterpret_cast<const float4*>(p)); b = __ldcs(reinterpret_cast<const float4*>(p) + 1); }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const {
    const __nv_bfloat162 u[4] = {__floats2bfloat162_rn(a.x, a.y), __floats2bfloat162_rn(a.z, a.w), __floats2bfloat162_rn(b.x, b.y),
                                 __floats2bfloat162_rn(b.z, b.w)};
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(u);
  }
};
template <> struct Pack<__nv_bfloat16, float, 4> {
  uint2 x;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { x = __ldcs(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ void store(float* p) const {
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x.x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x.y));
    *reinterpret_cast<float4*>(p) = make_float4(a.x, a.y, b.x, b.y);
  }
};

constexpr int ST_WARPS = 8;
template <typename S, typename D, int VEC>
__global__ void __launch_bounds__(ST_WARPS * 32)
kv_store_kernel(const S* __restrict__ k, const S* __restrict__ v, long long layer_k, long long layer_v, long long ld_k, long long ld_v,
                const int* __restrict__ row_map, D* __restrict__ k_pages, D* __restrict__ v_pages, int T, int n_pages, int KV, int hd) {
  tlc_wait(k, v, row_map, k_pages, v_pages);
  const int t = blockIdx.x * ST_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= T) return;
  const int place = row_map[t];
  if (place < 0 || place / TLC_PAGE >= n_pages) return;
  const int l = blockIdx.y, C = KV * hd;
  const size_t page = ((size_t)l * n_pages + place / TLC_PAGE) * KV;
  const size_t inside = (size_t)(place % TLC_PAGE) * hd;
  const S* kr = k + l * layer_k + t * ld_k;
  const S* vr = v ? v + l * layer_v + t * ld_v : nullptr;
  constexpr int U = 2;                                 // pieces a lane has on their way at a time
  for (int c0 = lane * VEC; c0 < C; c0 += U * 32 * VEC) {
    Pack<S, D, VEC> a[U], b[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = c0 + u * 32 * VEC;
      if (c < C) {
        a[u].load(kr + c);
        if (vr) b[u].load(vr + c);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int c = c0 + u * 32 * VEC;
      if (c < C) {
        const size_t to = (page + c / hd) * (size_t)(TLC_PAGE * hd) + inside + c % hd;
        a[u].store(k_pages + to);
        if (vr) b[u].store(v_pages + to);
      }
    }
  }
}

template <typename S, typename D>
void run_store(const void* k, const void* v, long long layer_k, long long layer_v, long long ld_k, long long ld_v, const int* row_map,
               void* k_pages, void* v_pages, int L, int T, int n_pages, int KV, int hd, cudaStream_t stream) {
  constexpr int WIDE = 16 / sizeof(D);
  const uintptr_t src = (uintptr_t)k | (uintptr_t)v | (uintptr_t)(layer_k * (long long)sizeof(S)) | (uintptr_t)(layer_v * (long long)sizeof(S)) |
                        (uintptr_t)(ld_k * (long long)sizeof(S)) | (uintptr_t)(ld_v * (long long)sizeof(S));
  const uintptr_t dst = (uintptr_t)k_pages | (uintptr_t)v_pages;
  const dim3 grid((T + ST_WARPS - 1) / ST_WARPS, L), block(ST_WARPS * 32);
  // whole pieces of 16 bytes where every row starts on such a boundary and a head is whole pieces
  if (hd % WIDE == 0 && (src % (sizeof(S) == 2 && sizeof(D) == 4 ? 8 : 16)) == 0 && dst % 16 == 0)
    tlc_launch(kv_store_kernel<S, D, WIDE>, grid, block, 0, stream, (const S*)k, (const S*)v, layer_k, layer_v, ld_k, ld_v, row_map,
               (D*)k_pages, (D*)v_pages, T, n_pages, KV, hd);
  else
    tlc_launch(kv_store_kernel<S, D, 1>, grid, block, 0, stream, (const S*)k, (const S*)v, layer_k, layer_v, ld_k, ld_v, row_map,
               (D*)k_pages, (D*)v_pages, T, n_pages, KV, hd);
}

}  // namespace

extern "C" int tlc_page_resize(int* block_table, int n_slots, int max_pages, int* refs, int n_pages, int* lengths, const int* slots,
                               const int* want, int B, int* status, cudaStream_t stream) {
  if (B == 0) return 0;
  TLC_REQUIRE(B > 0 && B <= MAX_REQUESTS, "page_resize: %d requests (at most %d a call)", B, MAX_REQUESTS);
  TLC_REQUIRE(n_slots > 0 && max_pages > 0 && n_pages > 0 && n_pages <= (1 << 25), "page_resize: %d slots of %d pages, %d pages (at most 2^25)",
              n_slots, max_pages, n_pages);
  // (the kernel adds up pages taken, and pages given back, in 32 bits each; slots are distinct)
  TLC_REQUIRE((long long)(B < n_slots ? B : n_slots) * max_pages < (1ll << 31), "page_resize: %d requests of up to %d pages, 2^31 or more together",
              B < n_slots ? B : n_slots, max_pages);
  static OncePerDevice ready;
  constexpr int most = (RT * PER + 2 * (MAX_REQUESTS + 1)) * (int)sizeof(int) + MAX_REQUESTS * (int)sizeof(Request);
  if (!ready.done([&] { return cudaFuncSetAttribute(page_resize_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most); }))
    return tlc_fail(-2, "page_resize: cannot reserve shared memory");
  const int smem = (RT * PER + 2 * (B + 1)) * (int)sizeof(int) + B * (int)sizeof(Request);
  tlc_launch(page_resize_kernel, dim3(1), dim3(RT), (size_t)smem, stream, block_table, n_slots, max_pages, refs, n_pages, lengths, slots, want, B,
             status);
  TLC_CHECK_LAUNCH("page_resize");
  return 0;
}

extern "C" int tlc_row_maps(const int* block_table, int n_slots, int max_pages, const int* slots, const int* lengths, const int* start,
                            const int* rows, int B, int T, const int* parents, const void* keep, int words, int* cu_seqlens, int* row_seq, int* positions,
                            int* row_map, int* mask, cudaStream_t stream) {
  TLC_REQUIRE(B >= 0 && B <= MAX_REQUESTS, "row_maps: %d requests (at most %d a call)", B, MAX_REQUESTS);
  TLC_REQUIRE(T >= 0 && n_slots > 0 && max_pages > 0 && (T == 0 || (parents == nullptr) == (mask == nullptr)) && words >= 0, "row_maps: %d rows, %d slots of %d pages",
              T, n_slots, max_pages);
  if (!mask) words = 0;
  tlc_launch(row_maps_kernel, dim3(T > 0 ? (T + MT - 1) / MT : 1), dim3(MT), (size_t)(B + 1) * sizeof(int), stream, block_table, n_slots, max_pages,
             slots, lengths, start, rows, B, T, parents, (const unsigned char*)keep, words, cu_seqlens, row_seq, positions, row_map, mask);
  TLC_CHECK_LAUNCH("row_maps");
  return 0;
}

extern "C" int tlc_kv_store(const void* k, const void* v, int dtype, long long layer_k, long long layer_v, long long ld_k, long long ld_v,
                            const int* row_map, void* k_pages, void* v_pages, int page_dtype, int L, int T, int n_pages, int KV, int hd,
                            cudaStream_t stream) {
  if (L == 0 || T == 0) return 0;
  TLC_REQUIRE(L > 0 && L <= 65535 && T > 0 && n_pages > 0 && n_pages <= (1 << 25) && KV > 0 && hd > 0 && (long long)KV * hd <= (1 << 30),
              "kv_store: %d layers, %d rows, %d pages, %d heads of %d", L, T, n_pages, KV, hd);
  TLC_REQUIRE((v == nullptr) == (v_pages == nullptr), "kv_store: values and their pages come together");
  TLC_DISPATCH_DTYPE(dtype, S, {
    TLC_DISPATCH_DTYPE(page_dtype, D, {
      run_store<S, D>(k, v, layer_k, layer_v, ld_k, ld_v, row_map, k_pages, v_pages, L, T, n_pages, KV, hd, stream);
    });
  });
  TLC_CHECK_LAUNCH("kv_store");
  return 0;
}
