// Products in 8-bit integers: out[m, n] (+)= a_scale[m] w_scale[n] sum_k a[m, k] w[n, k] + colbias[n], also gated (silu(gate) * up and
// the like) and grouped by expert.  The sum of integers is exact in 32 bits while K <= 131,071 (128 * 128 * K < 2^31), so neither the
// order of a sum nor how K is cut changes a result.
//
// The kernels, chosen in run() and tlc_linear_int8() by sizes, types and alignment alone:
//   gemm_int8_skinny.cu  one row (two that are to be rounded), and experts of up to 8 pairs: CUDA cores, rows rounded in the same kernel
//   gemm_int8_thin.cu    up to 16 rows of up to 4,096 values: mma.sync on weights that come from HBM into registers
//   gemm_int8_few.cu     up to 64 rows, more where tiles are few: tensor cores, K shared among the blocks of a cluster
//   gemm_int8_wide.cu    many rows, groups of 25 and more: tensor cores, pairs of blocks, persistent
//   here                 operands that the copy engine does not take (rows off 16-byte boundaries; gated outputs that are no multiple of
//                        8): CUDA cores (dp4a: four products and their sum an instruction), tiles of 32 x 64 results staged
//                        through shared memory 64 values of K at a time.  2,048 rows of 2,048 -> 8,240 956 us, 72 TOP/s, bound by
//                        shared memory (three reads for eight dp4a); the tensor cores take 31.
//
// Results added to what is there, as a model's projections back into the 32-bit stream are, cost little in the kernels of few rows
// and much in the pairs' (the old values of a piece are asked for when its sums are there).  Microseconds added, and written in 32 bits:
// 12 x 4,096 -> 2,048 3.3, 3.1; 64 rows 6.4, 6.3; 512 rows 12.7, 11.0; 2,048 rows 27.2, 17.1; 2,048 x 8,192 -> 2,560 56.8, 45.2; 8,192 rows 146,
// 134; 2,048 x 2,048 -> 8,240 82.6, 32.9.
#include "gemm_int8_tc.cuh"
#include <algorithm>
#include <atomic>

int tlc_rows_int8_pairs(const void* x, int x_dtype, int ldx, int T, int K, void* q, int ldq, float* scale, const int* order, int top, int* place,
                        cudaStream_t stream);       // int8_rows.cu
int tlc_int8_few(const Int8Args& p, int out_dtype, int nb, int sms, cudaStream_t stream);      // gemm_int8_few.cu
int tlc_int8_few_split(long long tiles, int num_k, int sms);
int tlc_int8_skinny(const void* x, int x_dtype, const Int8Args& p, int out_dtype, int sms, cudaStream_t stream);   // gemm_int8_skinny.cu
int tlc_int8_skinny_pairs(const void* x, int x_dtype, const Int8Args& p, const int* ids, int per_row, int out_dtype, int sms, cudaStream_t stream);
int tlc_int8_thin(const Int8Args& p, int out_dtype, cudaStream_t stream);                        // gemm_int8_thin.cu
int tlc_int8_wide(const Int8Args& p, int out_dtype, int nb, int pairs, cudaStream_t stream);   // gemm_int8_wide.cu

namespace {

constexpr int TM = 32, TN = 64, TKW = 16;          // a tile's rows and columns; K in words of four values

// Four values from k on as one word, zeros past K.
__device__ __forceinline__ int word_at(const int8_t* p, int k, int K, bool words) {
  if (words && k + 4 <= K) return *reinterpret_cast<const int*>(p + k);
  int v = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) if (k + i < K) v |= (int)(uint8_t)p[k + i] << (8 * i);
  return v;
}

template <typename TO, bool GLU>
__global__ void __launch_bounds__(256)
int8_tile_kernel(Int8Args p) {
  tlc_pdl(p.a, p.a_scale, p.w, p.out, p.offsets, p.order, p.wts);
  constexpr int NW = GLU ? 2 : 1;
  __shared__ int As[TM][TKW + 1], Ws[NW][TN][TKW + 1];
  const int tid = threadIdx.x, n0 = blockIdx.y * TN;
  int group = 0, row0, rows;
  if (p.offsets) {                                  // which group's tile this is: the tiles before it are counted
    int tile = blockIdx.x;
    bool found = false;
    for (; group < p.E; group++) {
      const int count = p.offsets[group + 1] - p.offsets[group], tiles = (count + TM - 1) / TM;
      if (tile < tiles) { found = true; break; }
      tile -= tiles;
    }
    if (!found) return;
    row0 = p.offsets[group] + tile * TM;
    rows = min(TM, p.offsets[group + 1] - row0);
  } else {
    row0 = blockIdx.x * TM;
    rows = min(TM, p.M - row0);
  }
  const bool words_a = ((uintptr_t)p.a | (uintptr_t)p.lda) % 4 == 0, words_w = ((uintptr_t)p.w | (uintptr_t)p.ldw) % 4 == 0;
  const size_t w0 = (size_t)group * p.w_rows;
  const int r2 = (tid >> 4) * 2, c0 = tid & 15;     // this thread's rows r2, r2 + 1 and columns c0 + 16 j
  int acc[NW][2][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += 4 * TKW) {
#pragma unroll
    for (int i = 0; i < TM * TKW / 256; i++) {
      const int r = (tid >> 4) + i * 16, k = k0 + 4 * (tid & 15);
      As[r][tid & 15] = r < rows ? word_at(p.a + (size_t)(row0 + r) * p.lda, k, p.K, words_a) : 0;
    }
#pragma unroll
    for (int u = 0; u < NW; u++)
#pragma unroll
      for (int i = 0; i < TN * TKW / 256; i++) {
        const int n = (tid >> 4) + i * 16, k = k0 + 4 * (tid & 15);
        Ws[u][n][tid & 15] = n0 + n < p.N ? word_at(p.w + (w0 + (size_t)u * p.N + n0 + n) * p.ldw, k, p.K, words_w) : 0;
      }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < TKW; k++) {
      const int a0 = As[r2][k], a1 = As[r2 + 1][k];
#pragma unroll
      for (int u = 0; u < NW; u++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int b = Ws[u][c0 + 16 * j][k];
          acc[u][0][j] = __dp4a(a0, b, acc[u][0][j]);
          acc[u][1][j] = __dp4a(a1, b, acc[u][1][j]);
        }
    }
    __syncthreads();
  }
  TO* out = reinterpret_cast<TO*>(p.out);
#pragma unroll
  for (int i = 0; i < 2; i++) {
    if (r2 + i >= rows) continue;
    const int row = row0 + r2 + i, pair = p.order ? p.order[row] : row;
    float rs = p.a_scale[row];
    if (p.w_out) rs *= p.wts[pair];
    const float pw = p.w_in ? p.wts[pair] : 1.0f;
    TO* o = out + (size_t)(p.scatter ? pair : row) * p.ldo;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int n = n0 + c0 + 16 * j;
      if (n >= p.N) continue;
      float v = int8_value(acc[0][i][j], rs, p.w_scale[w0 + n], p.colbias ? p.colbias[n] : 0.f);
      if (GLU || p.mode == I8_ACT) {
        float u = 0.f;
        if (GLU)
          u = int8_value(acc[NW - 1][i][j], rs, p.w_scale[w0 + p.N + n], p.colbias ? p.colbias[p.N + n] : 0.f);
        v = int8_gated(p, p.w_in, pw, v, u);
      } else if (p.mode == I8_ADD) {
        v += to_f32(o[n]);
      }
      o[n] = from_f32<TO>(v);
    }
  }
}

template <typename TO>
int run_tiles(const Int8Args& p, cudaStream_t stream) {
  // grouped: an upper bound, the last blocks find no tile
  const int tiles = p.offsets ? p.M / TM + (p.M < p.E ? p.M : p.E) : (p.M + TM - 1) / TM;
  const dim3 grid(tiles, (p.N + TN - 1) / TN);
  if (p.mode == I8_GLU) tlc_launch(int8_tile_kernel<TO, true>, grid, dim3(256), 0, stream, p);
  else tlc_launch(int8_tile_kernel<TO, false>, grid, dim3(256), 0, stream, p);
  TLC_CHECK_LAUNCH("linear_int8");
  return 0;
}

// Whether the copy engine takes the operands: rows that start on 16-byte boundaries, and gated weights whose rows come in eights.
bool tensor_cores_take(const Int8Args& p) {
  return ((uintptr_t)p.a | (uintptr_t)p.w | (uintptr_t)p.lda | (uintptr_t)p.ldw) % 16 == 0 && (p.mode != I8_GLU || p.N % 8 == 0) &&
         tlc_error_words_here() != nullptr;
}

int sm_count() {                     // (of the device that is asked first: it sizes grids, no more)
  static std::atomic<int> sms{0};
  if (sms == 0) {
    int dev = 0, n = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    sms = n > 0 ? n : 148;
  }
  return sms;
}

int g_kernel = 0, g_rows = 0;        // test hook: which kernel, on tiles of how many activation rows

int run(const Int8Args& p, int out_dtype, cudaStream_t stream) {
  const int sms = sm_count();
  // Up to 16 rows: weights straight to the registers of mma.sync, for one wave of blocks before the wait.  Microseconds there and through
  // shared memory, 8 rows: 2,048 -> 2,048 2.1, 3.6; 4,096 -> 2,048 2.5, 4.4; 2,048 -> 8,240 3.9, 6.0; 2,560 -> 2 x 8,192 9.2, 10.1;
  // 2,048 -> 65,536 22.6, 26.1.  12 rows: 2,048 -> 2,048 2.8, 3.7; 4,096 -> 2,048 3.2, 4.5; 2,048 -> 8,240 5.1, 6.1, but from 24 MB of
  // weights on 2,560 -> 10,240 8.2, 8.1; 2,560 -> 2 x 8,192 12.0, 10.2; 2,048 -> 65,536 30.8, 26.3.  (8 rows of 8,192 -> 2,560 by clusters
  // of two blocks 7.6, 6.8.)
  const bool thin = p.M <= 8 || (p.M <= 16 && (long long)p.w_rows * p.K <= 24 << 20);
  if (!p.offsets && (g_kernel == 5 ? p.M <= 16 : thin && (g_kernel == 0 || g_kernel == 4)) && p.K <= TLC_INT8_THIN &&
      ((uintptr_t)p.w | (uintptr_t)p.ldw) % 16 == 0)
    return tlc_int8_thin(p, out_dtype, stream);
  if (g_kernel != 1 && tensor_cores_take(p)) {
    const int pairs = p.ldo < 1 << 27 ? tlc_linear_pairs() : 0;      // (sixteen rows of a result are addressed in 32 bits there)
    if (g_kernel == 3 && pairs > 0) return tlc_int8_wide(p, out_dtype, g_rows, pairs, stream);
    if (g_kernel == 2) return tlc_int8_few(p, out_dtype, g_rows, sms, stream);
    if (p.offsets) {
      // Rows of a group, on average.  From 25 on pairs of blocks, which stay and stream through the groups one after the other; microseconds
      // of a whole feed-forward with tiles of 128 rows by single blocks, of 128 and of 256 rows by pairs: 25 rows (32 experts) 61, 56, 60;
      // 73 rows (64 experts) 129, 88, 99; 188 rows (32 experts) 151, 99, 84.  Below, 5 rows (32 experts) 48 with tiles of 16, 51 by pairs.
      const int rows = (p.M + p.E - 1) / p.E, most = rows * 3 / 2;         // (a group may well have half as many again)
      if (pairs > 0 && rows > 24) return tlc_int8_wide(p, out_dtype, rows <= 110 ? 128 : 256, pairs, stream);
      return tlc_int8_few(p, out_dtype, most <= 16 ? 16 : most <= 32 ? 32 : most <= 64 ? 64 : 128, sms, stream);
    }
    if (p.M <= 64) return tlc_int8_few(p, out_dtype, p.M <= 16 ? 16 : p.M <= 32 ? 32 : 64, sms, stream);
    // More rows: whichever of three is through first by what a K-step and the way in and out take (microseconds, measured): tiles of 64
    // or 128 rows by single blocks that share K, where the tiles are few, or tiles of 256 rows by pairs.  For 129, 512 and 1,031 rows
    // (64, 128, pairs): 2,560 -> 1,537 6.3 8.5 10.5, 9.1 9.4 11.5, 12.9 12.3 11.6; 8,192 -> 2,560 10.9 13.3 23.2, 25.9 19.6 24.3,
    // 49.9 32.4 25.8; 2,048 -> 8,240 11.7 11.2 9.7, 23.4 17.0 12.7, 45.5 33.7 23.9.
    const int num_k = (p.K + I8_K - 1) / I8_K, w_rows = p.mode == I8_GLU ? 2 * p.N : p.N;
    auto single = [&](int nb, float way, float step) {
      const long long tiles = (long long)((w_rows + I8_ROWS - 1) / I8_ROWS) * ((p.M + nb - 1) / nb);
      const int split = tlc_int8_few_split(tiles, num_k, sms);
      return way + step * (float)((tiles * split + 2 * sms - 1) / (2 * sms) * ((num_k + split - 1) / split));
    };
    const float by64 = single(64, 4.7f, 0.36f), by128 = single(128, 6.5f, 0.46f);
    if (pairs > 0) {
      const long long tiles = (long long)((w_rows + 2 * I8_ROWS - 1) / (2 * I8_ROWS)) * ((p.M + 255) / 256);
      if (4.6f + 0.32f * (float)((tiles + pairs - 1) / pairs * num_k) <= std::min(by64, by128)) return tlc_int8_wide(p, out_dtype, 256, pairs, stream);
    }
    return tlc_int8_few(p, out_dtype, by64 <= by128 ? 64 : 128, sms, stream);
  }
  return out_dtype == TLC_F32 ? run_tiles<float>(p, stream) : run_tiles<__nv_bfloat16>(p, stream);
}

}  // namespace

// Test hook: 0 = chosen by the sizes; 1 = the CUDA cores; 2 = tiles of 128 weight rows and 16, 32, 64 or 128 activation rows; 3 = pairs of
// blocks on 256 weight rows and 128 or 256 activation rows; 4 = the kernel of one or two rows; 5 = the kernel of up to 16 rows, wherever
// they take the operands.
extern "C" int tlc_linear_int8_kernel(int kernel, int rows) {
  TLC_REQUIRE(kernel == 0 || kernel == 1 || (kernel == 2 && (rows == 16 || rows == 32 || rows == 64 || rows == 128)) ||
              (kernel == 3 && (rows == 128 || rows == 256)) || kernel == 4 || kernel == 5, "linear_int8: there is no kernel %d with tiles of %d rows", kernel, rows);
  g_kernel = kernel;
  g_rows = rows;
  return 0;
}

extern "C" int tlc_linear_int8(const void* a, int a_dtype, int lda, float* a_scale, void* a_int8, int ld_int8, const void* w, int ldw,
                               const float* w_scale, void* out, int out_dtype, int ldo, const float* colbias, int accumulate, int M, int N,
                               int K, int act, float limit, float alpha, cudaStream_t stream) {
  if (M == 0 || N == 0) return 0;
  TLC_REQUIRE(K > 0 && K <= 131071 && lda >= K && ldw >= K && ldo >= N && M > 0 && N > 0,
              "linear_int8: bad sizes M=%d N=%d K=%d (at most 131071) lda=%d ldw=%d ldo=%d", M, N, K, lda, ldw, ldo);
  TLC_REQUIRE(act < 0 || act == TLC_ACT_SILU || act == TLC_ACT_GELU_TANH || act == TLC_ACT_SWISH_CLAMPED, "linear_int8: unknown activation %d", act);
  Int8Args p = {};
  p.a = (const int8_t*)a; p.a_scale = a_scale; p.w = (const int8_t*)w; p.w_scale = w_scale; p.out = out; p.colbias = colbias;
  p.lda = lda; p.ldw = ldw; p.ldo = ldo; p.M = M; p.N = N; p.K = K; p.w_rows = act >= 0 ? 2 * N : N;
  p.mode = act >= 0 ? I8_GLU : accumulate ? I8_ADD : I8_PLAIN;
  p.act = act; p.limit = limit; p.alpha = alpha;
  TLC_REQUIRE(a_dtype == TLC_I8 || a_dtype == TLC_F32 || a_dtype == TLC_BF16, "linear_int8: unknown type %d of the rows", a_dtype);
  TLC_REQUIRE(out_dtype == TLC_F32 || out_dtype == TLC_BF16, "linear_int8: unknown output dtype %d", out_dtype);
  // One row of at most 8,192 values, weights in 16-byte pieces and up to 24 MB of them: the kernel that takes the row as it is.
  // Microseconds there and by gemm_int8_thin.cu (from K = 4,097 the tensor cores), a row to be rounded: 2,048 -> 2,048 2.1, 2.8; 2,048 ->
  // 8,240 3.7, 4.5; 4,096 -> 2,048 3.0, 3.5; 2,048 -> 2 x 4,096 3.4, 4.6; 8,192 -> 2,560 7.4, 7.5; 2,560 -> 10,240 8.2, 6.8.  Integers
  // behind the norm that makes them, both: 2,048 -> 8,240 4.5, 4.8; gated 4.5, 5.0.  Two rows that are to be rounded, up to K = 2,048: 2,048
  // -> 2,048 2.9, 3.1, -> 8,240 4.5, 4.5, and a launch less for the host (4,096 -> 2,048 4.6, 3.7; three rows 6.8, 4.6).
  const bool takes = (M == 1 ? K <= TLC_INT8_SKINNY : M == 2 && a_dtype != TLC_I8 && K <= TLC_INT8_TWO) && ((uintptr_t)w | (uintptr_t)ldw) % 16 == 0;
  if (takes && (g_kernel == 4 || (g_kernel == 0 && (long long)p.w_rows * K <= 24 << 20))) return tlc_int8_skinny(a, a_dtype, p, out_dtype, sm_count(), stream);
  if (a_dtype != TLC_I8) {
    if (!a_int8 || !a_scale) return 1;                     // (room is wanted)
    if (int rc = tlc_rows_int8(a, a_dtype, lda, M, K, nullptr, 0.f, a_int8, ld_int8, a_scale, nullptr, 1, 0, stream)) return rc;
    p.a = (const int8_t*)a_int8;
    p.lda = ld_int8;
  }
  return run(p, out_dtype, stream);
}

extern "C" int tlc_moe_experts_int8(const void* x, int x_dtype, int ldx, const void* wgu, int ldgu, const float* sgu, const void* wd, int ldd,
                                    const float* sd, const int* ids, const int* order, const int* offsets, const float* wts, int T, int E, int top, int F,
                                    int D, void* q, int ldq, float* scales, float* act, void* y, int y_dtype, int act_code, int w_out,
                                    float limit, float alpha, cudaStream_t stream) {
  if (T == 0) return 0;
  const long long pairs = (long long)T * top;
  TLC_REQUIRE(T > 0 && top >= 1 && E >= 1 && F >= 1 && D >= 1 && F <= 131071 && D <= 131071 && pairs < (1 << 30),
              "moe_experts_int8: bad sizes T=%d E=%d top=%d F=%d D=%d", T, E, top, F, D);
  TLC_REQUIRE(E <= TLC_INT8_GROUPS, "moe_experts_int8: %d experts (at most %d)", E, TLC_INT8_GROUPS);
  TLC_REQUIRE(ldgu >= D && ldd >= F && ldq >= D && ldq >= F, "moe_experts_int8: rows shorter than the sizes (ld %d %d %d)", ldgu, ldd, ldq);
  TLC_REQUIRE(act_code >= TLC_ACT_SILU && act_code <= TLC_ACT_RELU_SQUARED, "moe_experts_int8: unknown activation %d", act_code);
  TLC_REQUIRE((x_dtype == TLC_F32 || x_dtype == TLC_BF16) && (y_dtype == TLC_F32 || y_dtype == TLC_BF16), "moe_experts_int8: unknown dtype %d or %d",
              x_dtype, y_dtype);
  const bool gated = act_code != TLC_ACT_RELU_SQUARED;
  Int8Args p = {};
  p.a = (const int8_t*)q; p.a_scale = scales; p.w = (const int8_t*)wgu; p.w_scale = sgu; p.out = act;
  p.lda = ldq; p.ldw = ldgu; p.ldo = F; p.M = (int)pairs; p.N = F; p.K = D; p.w_rows = gated ? 2 * F : F;
  p.mode = gated ? I8_GLU : I8_ACT; p.act = act_code; p.limit = limit; p.alpha = alpha;
  p.offsets = offsets; p.order = order; p.wts = wts; p.E = E; p.w_in = !w_out;
  Int8Args d = p;                                         // the second product
  d.w = (const int8_t*)wd; d.w_scale = sd; d.out = y; d.ldw = ldd; d.ldo = D; d.N = D; d.K = F; d.w_rows = D;
  d.mode = I8_PLAIN; d.w_in = 0; d.w_out = w_out; d.scatter = 1;
  // A few pairs: each a product of one row, which the kernel rounds itself.  Microseconds there and in the four launches below (2,048 x
  // 1,024, 32 experts): 4 pairs 11.8, 16.2; 8 pairs 17.2, 19.2; 12 pairs 23.1, 23.0
  if ((g_kernel == 0 || g_kernel == 4) && pairs <= 8 && D <= TLC_INT8_SKINNY && F <= TLC_INT8_SKINNY &&
      ((uintptr_t)wgu | (uintptr_t)wd | (uintptr_t)ldgu | (uintptr_t)ldd) % 16 == 0) {
    p.lda = ldx;
    d.lda = F;
    if (int rc = tlc_int8_skinny_pairs(x, x_dtype, p, ids, top, TLC_F32, sm_count(), stream)) return rc;
    return tlc_int8_skinny_pairs(act, TLC_F32, d, ids, 1, y_dtype, sm_count(), stream);
  }
  // the chosen rows, sorted by expert, rounded; both products read their rows from q
  // (the activation's place has not been written yet and lends itself to the pairs' places)
  if (int rc = tlc_rows_int8_pairs(x, x_dtype, ldx, T, D, q, ldq, scales, order, top, (int*)act, stream)) return rc;
  if (int rc = run(p, TLC_F32, stream)) return rc;
  // the activation in 32 bits -> rounded row by row; a weight on the result only multiplies the row's scale
  if (int rc = tlc_rows_int8(act, TLC_F32, F, (int)pairs, F, nullptr, 0.f, q, ldq, scales, nullptr, 1, 0, stream)) return rc;
  return run(d, y_dtype, stream);
}
