// Eviction from a KV cache by accumulated attention weight: the weight that rows collect in prompts (that of decode steps is
// added up where it is pooled, in decode.cu), the choice of the rows that stay, and the moves that bring them together.  The
// declarations in kascade_b200.h say what each entry point computes; the reference has no counterpart.
#include <cooperative_groups.h>

#include <cfloat>
#include <climits>

#include "common.cuh"

namespace kb200 {

// ---- weight of a prompt ----------------------------------------------------------------------------------------------
struct PromptMassParams {
  const float* pooled; int64_t row_stride;
  const int32_t* seq_len;
  const float* mass_in; float* mass_out; int64_t in_stride, out_stride;
  int G, T, n_rows;
};

// 256 rows of the cache, twice four per lane, are a block; the pooled scores of a block are one piece of 1024 bytes per head and later
// tile, which a cluster of CTAs deals to its warps, four pieces in flight each.  The first rows have the most later tiles and the
// last none, so a cluster takes the i-th block from the front and the i-th from the back: equal work everywhere.  A lane
// adds its pieces up one after the other, the warps' and the CTAs' sums meet in the order of their numbers, so a call
// gives the same bits every time.  us with 128 / 256 / 512 rows in a block: one prompt of 32768 rows 94.6 / 90.9 / 88.3, 16384 30.6 / 28.7
// / 35.8, 8192 13.6 / 14.6 / 19.8, 8 x 4096 18.8 / 17.8 / 18.7.
constexpr int kMassWarps = 16;
constexpr int kMassVec = 2;                                       // pieces of 512 bytes beside each other that a warp reads at once
constexpr int kMassUnroll = 4;
constexpr int kMassRows = 128 * kMassVec;                         // of a block
__global__ void __launch_bounds__(kMassWarps * 32) mass_prompt_kernel(const PromptMassParams p) {
  namespace cg = cooperative_groups;
  pdl_begin();
  __shared__ float4 sums[kMassWarps][kMassVec * 32];
  __shared__ float total[2][kMassRows];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tiles = p.seq_len ? min((max(p.seq_len[b], 0) + kTile - 1) / kTile, p.T) : p.T;
  const int blocks = (p.n_rows + kMassRows - 1) / kMassRows, front = blockIdx.x / ctas, back = blocks - 1 - front;
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    const int block = half ? back : front;
    const int j = block * kMassRows + lane * 4;
    const int first = block * (kMassRows / kTile) + 1;              // the first tile behind the first of these rows
    const int later = half && back == front ? 0 : max(tiles - first, 0), pieces = later * p.G, step = ctas * kMassWarps;
    const float* rows = p.pooled + (int64_t)b * p.G * p.T * p.row_stride + j;
    float4 a[kMassVec];
#pragma unroll
    for (int v = 0; v < kMassVec; ++v) a[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = rank * kMassWarps + warp; i0 < pieces; i0 += step * kMassUnroll) {
      float4 x[kMassUnroll][kMassVec];
#pragma unroll
      for (int u = 0; u < kMassUnroll; ++u) {
        const int i = i0 + u * step, g = i / later, t = first + i - g * later;
        const float* src = rows + ((int64_t)g * p.T + t) * p.row_stride;
#pragma unroll
        for (int v = 0; v < kMassVec; ++v) {
          x[u][v] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i < pieces && t > (j + v * 128) / kTile) x[u][v] = *reinterpret_cast<const float4*>(src + v * 128);
        }
      }
#pragma unroll
      for (int u = 0; u < kMassUnroll; ++u)
#pragma unroll
        for (int v = 0; v < kMassVec; ++v) { a[v].x += x[u][v].x; a[v].y += x[u][v].y; a[v].z += x[u][v].z; a[v].w += x[u][v].w; }
    }
#pragma unroll
    for (int v = 0; v < kMassVec; ++v) sums[warp][v * 32 + lane] = a[v];
    __syncthreads();
    for (int i = threadIdx.x; i < kMassRows; i += kMassWarps * 32) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kMassWarps; ++w) s += reinterpret_cast<const float*>(sums[w])[i];
      total[half][i] = s;
    }
    __syncthreads();
  }
  cluster.sync();
  if (rank == 0) {
    for (int i0 = threadIdx.x; i0 < kMassRows * (back == front ? 1 : 2); i0 += kMassWarps * 32) {
      const int half = i0 / kMassRows, at = i0 - half * kMassRows;
      float s = total[half][at];
      for (int r = 1; r < ctas; ++r) s += cluster.map_shared_rank(&total[0][0], r)[half * kMassRows + at];
      const int i = (half ? back : front) * kMassRows + at;
      if (i < p.n_rows) p.mass_out[b * p.out_stride + i] = p.mass_in[b * p.in_stride + i] + s;
    }
  }
  cluster.sync();                                                  // the sums have been read
}

// CTAs that share two blocks: doubled while all of them together are at most two per SM.  512 threads with eight loads each
// keep enough in flight then, and a second round of CTAs would leave SMs idle at its end (with blocks of 128 rows and at most two
// / four CTAs per SM: one prompt of 32768 rows 95 / 102 us, 16384 30.5 / 38.4, 8192 13.8 / 13.6, 8 x 4096 18.8 / 24.6, 4 x 3001 11.9 /
// 17.3).  32768 rows: 5.9 TB/s, 0.92 of the copy.  (A thread per four rows, over all heads and tiles: 1995 us.)
static int mass_ctas(int64_t clusters) {
  int c = 1;
  while (c < 8 && clusters * c <= sm_count()) c *= 2;
  return c;
}

// ---- what stays ------------------------------------------------------------------------------------------------------
// What the rows of a sequence are ranked by: +inf for protected ones, else their weight (a NaN counts as 0, an infinite one as the
// largest number, so that it stays behind the protected rows).  A cluster of CTAs
// takes a sequence: the newest position first, over all of it, then the keys of its piece.  Latency is what counts: 4 sequences of 32768
// rows 20.6 us with one CTA each, 7.8 with eight; counting the protected rows, where rows have positions of their own, takes 2 more.
// Rows that share a position (images on several axes) can be more than the budget holds.  Then the lowest `sinks` rows of the first
// positions get +inf, the recent ones a key that falls with their distance from the newest position, above all weights: the last
// `recent` rows in the order of positions stay in any case.  Only where the newest position alone has more rows than
// the budget do all protected rows count alike.
constexpr int kKeyThreads = 1024;
struct EvictKeysParams {
  const float* mass; int64_t mass_stride;
  const int32_t* seq_lens;
  const int32_t* positions; int64_t pos_stride;
  float* keys; int64_t key_stride;
  int sinks, recent, budget, n_rows;
};

// Sums of N numbers of each thread over the cluster.  All its threads call it.
template <int N>
__device__ __forceinline__ void cluster_sums(int (&v)[N], int (*of_warp)[32], int* of_cta) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = __reduce_add_sync(0xFFFFFFFFu, v[i]);
    if ((tid & 31) == 0) of_warp[i][tid >> 5] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = __reduce_add_sync(0xFFFFFFFFu, of_warp[i][tid & 31]);
    if (tid == 0) of_cta[i] = v[i];
  }
  cluster.sync();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0;
    for (int r = 0; r < (int)cluster.num_blocks(); ++r) v[i] += cluster.map_shared_rank(of_cta, r)[i];
  }
  cluster.sync();                                                 // the others have read this CTA's sums
}

__global__ void __launch_bounds__(kKeyThreads) evict_keys_kernel(const EvictKeysParams p) {
  namespace cg = cooperative_groups;
  pdl_begin();
  __shared__ int newest_of[32], newest_s, sums_of[2][32], sums_s[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x;
  const int b = blockIdx.x / ctas, n = min(p.seq_lens[b], p.n_rows);
  const int j0 = rank * kKeyThreads + tid, step = ctas * kKeyThreads;
  const float* mass = p.mass + b * p.mass_stride;
  const int32_t* positions = p.positions ? p.positions + b * p.pos_stride : nullptr;
  float* keys = p.keys + b * p.key_stride;
  auto weight = [&](int j, float most) { const float m = mass[j]; return m == m ? fminf(m, most) + 0.f : 0.f; };   // (-0 is 0)
  if (!positions) {
    for (int j = j0; j < n; j += step) keys[j] = j < p.sinks || j >= n - p.recent ? INFINITY : weight(j, FLT_MAX);
    return;
  }
  int newest = INT_MIN;
  for (int j = j0; j < n; j += step) newest = max(newest, positions[j]);
  newest = __reduce_max_sync(0xFFFFFFFFu, newest);
  if ((tid & 31) == 0) newest_of[tid >> 5] = newest;
  __syncthreads();
  newest = __reduce_max_sync(0xFFFFFFFFu, newest_of[tid & 31]);
  if (tid == 0) newest_s = newest;
  cluster.sync();
  for (int r = 0; r < ctas; ++r) newest = max(newest, *cluster.map_shared_rank(&newest_s, r));
  auto is_first = [&](int pos) { return pos >= 0 && pos < p.sinks; };          // (a negative one was never noted)
  auto is_recent = [&](int pos) { return (int64_t)pos > (int64_t)newest - p.recent; };
  int kept[1] = {0};
  for (int j = j0; j < n; j += step) {
    const int pos = positions[j];
    const bool stays = is_first(pos) || is_recent(pos);
    keys[j] = stays ? INFINITY : weight(j, FLT_MAX);
    kept[0] += stays;
  }
  cluster_sums(kept, sums_of, sums_s);
  if (kept[0] <= p.budget) return;                                // (the same for the whole cluster)
  int count[2] = {0, 0};                                          // rows of the newest position, of the first ones
  for (int j = j0; j < n; j += step) {
    count[0] += positions[j] == newest;
    count[1] += is_first(positions[j]);
  }
  cluster_sums(count, sums_of, sums_s);
  if (count[0] > p.budget) return;
  int end = n;                                                    // below it lie the first `sinks` rows of the first positions
  if (count[1] > p.sinks) {
    int lo = 0;
    while (lo < end) {
      const int mid = lo + (end - lo) / 2;
      int below[1] = {0};
      for (int j = j0; j < mid; j += step) below[0] += is_first(positions[j]);
      cluster_sums(below, sums_of, sums_s);
      if (below[0] >= p.sinks) end = mid;
      else lo = mid + 1;
    }
  }
  constexpr int kMost = 0x7F7FFFFF, kSteps = 0x7FFFFF;            // the largest number, and the numbers above 2^127
  for (int j = j0; j < n; j += step) {
    const int pos = positions[j];
    keys[j] = is_first(pos) && j < end ? INFINITY
              : is_recent(pos)         ? __int_as_float(kMost - (int)min((int64_t)newest - pos, (int64_t)kSteps))
                                       : weight(j, __int_as_float(kMost - kSteps - 1));
  }
}

struct EvictPlanParams {
  const int32_t* keep; int64_t keep_stride; const int32_t* keep_count;
  const float* mass_in; int64_t mass_stride;
  const int32_t* pos_in; int64_t pos_stride;
  int2* moves; int32_t* move_count; int32_t* new_lens;
  float* mass_out; int32_t* pos_out; int64_t out_stride;
  int n_rows;
};

// The first place of the ascending list a[0..n) whose value is not below x, by one warp: 32 probes at a time, four rounds for
// a million entries instead of twenty loads one after the other.
__device__ __forceinline__ int warp_lower_bound(const int32_t* a, int n, int x) {
  const int lane = threadIdx.x & 31;
  int lo = 0, len = n;                                            // the answer lies in [lo, lo + len]
  while (len > 0) {
    const int step = (len + 31) / 32, at = lo + lane * step;       // the last probe is the last of its piece, or beyond
    const int last = min(at + step, lo + len) - 1;
    const unsigned below = __ballot_sync(0xFFFFFFFFu, at < lo + len && a[max(last, 0)] < x);
    const int whole = __popc(below);                               // pieces that lie below x as a whole: a prefix
    const int end = lo + len;
    lo = min(lo + whole * step, end);
    len = min(step, end - lo);
    if (step == 1) len = 0;
  }
  return lo;
}

// A CTA takes 256 rows.  The rank of a row among the kept ones comes from a bitmap of the kept rows among the 256 and the rank of
// the first (with a binary search for every row 12.7 us for 4 x 32768 rows, so 6.5).  A row below the new length that is let go has
// i - rank others let go before it, and takes the (i - rank)-th of the kept rows behind the new length.
__global__ void __launch_bounds__(256) evict_plan_kernel(const EvictPlanParams p) {
  pdl_begin();
  __shared__ uint32_t kept[8];
  __shared__ int stay_s, rank_s;
  const int b = blockIdx.y, i0 = blockIdx.x * 256, tid = threadIdx.x, i = i0 + tid, warp = tid >> 5;
  const int left = p.keep_count[b];
  const int32_t* keep = p.keep + b * p.keep_stride;
  if (tid < 8) kept[tid] = 0u;
  if (warp < 2) {
    const int at = warp_lower_bound(keep, left, warp == 0 ? left : i0);
    if ((tid & 31) == 0) (warp == 0 ? stay_s : rank_s) = at;
  }
  __syncthreads();
  const int stay = stay_s, rank = rank_s;                          // kept rows below the new length; kept rows below i0
  if (rank + tid < left) {
    const int row = keep[rank + tid] - i0;
    if (row < 256) atomicOr(&kept[row >> 5], 1u << (row & 31));
  }
  __syncthreads();
  if (i >= p.n_rows) return;
  if (i == 0) {
    p.new_lens[b] = left;
    p.move_count[b] = left - stay;
  }
  float mass = 0.f;
  int pos = -1;
  if (i < left) {
    int from = i;
    if (!((kept[warp] >> (tid & 31)) & 1u)) {
      int r = rank + __popc(kept[warp] & ((1u << (tid & 31)) - 1u));
      for (int w = 0; w < warp; ++w) r += __popc(kept[w]);
      from = keep[stay + i - r];
      p.moves[b * p.keep_stride + i - r] = make_int2(from, i);
    }
    mass = p.mass_in[b * p.mass_stride + from];
    pos = p.pos_in ? p.pos_in[b * p.pos_stride + from] : from;
  }
  p.mass_out[b * p.out_stride + i] = mass;
  p.pos_out[b * p.out_stride + i] = pos;
}

// ---- the moves -------------------------------------------------------------------------------------------------------
constexpr int kMoveLayers = 32;                                    // layers of one launch (the parameters have to hold their addresses)
struct EvictMoveParams {
  uint8_t* k[kMoveLayers]; uint8_t* v[kMoveLayers];               // codes or 16-bit rows
  uint8_t* kp[kMoveLayers]; uint8_t* vp[kMoveLayers];             // parameters of an INT4 cache
  int64_t sb, sp, st, sh;                                          // bytes
  int64_t pb, pp, pt, ph;
  const int32_t* block_table; int bt_stride, page_shift, page_mask;
  const int2* moves; int64_t move_stride; const int32_t* move_count;
  int G, row_chunks;                                               // 16-byte pieces of a row: 16, or 4 of an INT4 cache
};

// One warp per move and layer, 16 bytes per lane and step: bound by HBM (32768 moves of 8 layers, 2.15 GB: 346 us, 6.2 TB/s).
__global__ void __launch_bounds__(256) evict_move_kernel(const __grid_constant__ EvictMoveParams p) {
  pdl_begin();
  const int b = blockIdx.z, layer = blockIdx.y, lane = threadIdx.x & 31;
  const int j = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (j >= p.move_count[b]) return;
  const int2 move = p.moves[b * p.move_stride + j];
  int64_t page[2], slot[2];
  const int rows[2] = {move.x, move.y};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int lp = rows[e] >> p.page_shift;
    slot[e] = rows[e] & p.page_mask;
    page[e] = p.block_table ? p.block_table[(int64_t)b * p.bt_stride + lp] : lp;
  }
  for (int what = 0; what < (p.kp[layer] ? 4 : 2); ++what) {
    const bool par = what >= 2;
    uint8_t* base = what == 0 ? p.k[layer] : what == 1 ? p.v[layer] : what == 2 ? p.kp[layer] : p.vp[layer];
    const int64_t from = b * (par ? p.pb : p.sb) + page[0] * (par ? p.pp : p.sp) + slot[0] * (par ? p.pt : p.st);
    const int64_t to = b * (par ? p.pb : p.sb) + page[1] * (par ? p.pp : p.sp) + slot[1] * (par ? p.pt : p.st);
    const int chunks = par ? 1 : p.row_chunks;
    for (int c = lane; c < p.G * chunks; c += 32) {
      const int64_t at = (c / chunks) * (par ? p.ph : p.sh) + (c % chunks) * 16;
      *reinterpret_cast<uint4*>(base + to + at) = *reinterpret_cast<const uint4*>(base + from + at);
    }
  }
}

}  // namespace kb200

extern "C" int kb200_mass_add_prompt(const float* pooled, int64_t row_stride, const int32_t* seq_len, const float* mass_in,
                                     float* mass_out, int64_t mass_in_stride, int64_t mass_out_stride, int batch,
                                     int num_kv_heads, int num_tiles, int n_rows, void* stream) {
  using namespace kb200;
  KB_ENTRY(pooled, "mass_add_prompt: pooled");
  KB_REQUIRE(pooled && mass_in && mass_out, "mass_add_prompt: null pointer");
  KB_REQUIRE(batch >= 0 && batch <= 65535 && num_kv_heads > 0 && num_tiles >= 0 && n_rows >= 0, "mass_add_prompt: bad sizes");
  const int64_t need = num_tiles > 0 ? (int64_t)(num_tiles - 1) * kTile : 0;
  KB_REQUIRE(row_stride % 4 == 0 && row_stride >= need && (reinterpret_cast<uintptr_t>(pooled) & 15) == 0,
             "mass_add_prompt: pooled rows must be 16-byte aligned (row_stride %% 4 == 0) and hold %lld scores", (long long)need);
  KB_REQUIRE(batch <= 1 || (mass_in_stride >= n_rows && mass_out_stride >= n_rows), "mass_add_prompt: rows of mass overlap");
  KB_REQUIRE(n_rows >= need, "mass_add_prompt: mass holds %d rows, %d tiles need %lld", n_rows, num_tiles, (long long)need);
  if (batch == 0 || n_rows == 0) return 0;
  PromptMassParams p{pooled, row_stride, seq_len, mass_in, mass_out, mass_in_stride, mass_out_stride, num_kv_heads, num_tiles, n_rows};
  const int clusters = ceil_div(n_rows, 2 * kMassRows), ctas = mass_ctas((int64_t)clusters * batch);
  KB_LAUNCH("mass_prompt_kernel", launch_pdl(mass_prompt_kernel, dim3(clusters * ctas, batch), kMassWarps * 32, 0, (cudaStream_t)stream,
                                             ctas, p));
  return 0;
}

namespace kb200 {
// the pieces of the workspace, in 4-byte words: keys [B, keys_row], kept rows [B, budget] and their count [B], moves [B, budget] pairs
// and their count [B]
struct EvictWorkspace {
  int64_t keys_row, keep, keep_count, moves, move_count, words;
  EvictWorkspace(int64_t batch, int64_t n_rows, int64_t budget) {
    keys_row = (n_rows + 3) / 4 * 4;
    moves = batch * keys_row;                                      // (8-byte aligned: a multiple of four words)
    keep = moves + 2 * batch * budget;
    keep_count = keep + batch * budget;
    move_count = keep_count + batch;
    words = move_count + batch;
  }
};

static int check_layers(const kb200_kv_layout* layers, int n_layers) {
  const kb200_kv_layout& one = layers[0];
  const bool int4 = one.dtype == KB200_INT4;
  KB_REQUIRE(one.dtype == KB200_FP16 || one.dtype == KB200_BF16 || int4,
             "evict: fp16, bf16 or INT4 caches (dtype code %d): an FP8 row is stored in the scale of its page and cannot leave it",
             one.dtype);
  KB_REQUIRE(one.page_size >= 1 && (one.page_size & (one.page_size - 1)) == 0,
             "evict: page_size must be a power of two (got %d)", one.page_size);
  for (int i = 0; i < n_layers; ++i) {
    const kb200_kv_layout& l = layers[i];
    KB_REQUIRE(l.k && l.v, "evict: null cache of layer %d", i);
    KB_REQUIRE(l.dtype == one.dtype && l.page_size == one.page_size && l.block_table == one.block_table &&
                   l.block_table_stride == one.block_table_stride && l.stride_batch == one.stride_batch &&
                   l.stride_page == one.stride_page && l.stride_token == one.stride_token && l.stride_head == one.stride_head &&
                   (!int4 || (l.param_stride_batch == one.param_stride_batch && l.param_stride_page == one.param_stride_page &&
                              l.param_stride_token == one.param_stride_token && l.param_stride_head == one.param_stride_head)),
               "evict: layer %d has another type, block table or strides than layer 0", i);
    KB_REQUIRE(((reinterpret_cast<uintptr_t>(l.k) | reinterpret_cast<uintptr_t>(l.v)) & 15) == 0 &&
                   ((l.stride_batch | l.stride_page | l.stride_token | l.stride_head) & (int4 ? 15 : 7)) == 0,
               "evict: caches must be 16-byte aligned, with strides that are multiples of 16 bytes");
    if (int4 && check_int4(&l, true, "evict") != 0) return -1;
  }
  return 0;
}

static int move_rows(const kb200_kv_layout* layers, int n_layers, const int2* moves, int64_t move_stride, const int32_t* move_count,
                     int max_moves, int batch, int num_kv_heads, cudaStream_t st) {
  const kb200_kv_layout& one = layers[0];
  const bool int4 = one.dtype == KB200_INT4;
  EvictMoveParams p{};
  const int64_t unit = int4 ? 1 : 2;
  p.sb = one.stride_batch * unit; p.sp = one.stride_page * unit; p.st = one.stride_token * unit; p.sh = one.stride_head * unit;
  p.pb = one.param_stride_batch * 2; p.pp = one.param_stride_page * 2; p.pt = one.param_stride_token * 2; p.ph = one.param_stride_head * 2;
  p.block_table = one.block_table;
  p.bt_stride = one.block_table_stride;
  int shift = 0;
  while ((1 << shift) < one.page_size) ++shift;
  p.page_shift = shift;
  p.page_mask = one.page_size - 1;
  p.moves = moves;
  p.move_stride = move_stride;
  p.move_count = move_count;
  p.G = num_kv_heads;
  p.row_chunks = int4 ? kD / 2 / 16 : kD * 2 / 16;
  for (int first = 0; first < n_layers; first += kMoveLayers) {
    const int n = n_layers - first < kMoveLayers ? n_layers - first : kMoveLayers;
    for (int i = 0; i < n; ++i) {
      const kb200_kv_layout& l = layers[first + i];
      p.k[i] = static_cast<uint8_t*>(const_cast<void*>(l.k));
      p.v[i] = static_cast<uint8_t*>(const_cast<void*>(l.v));
      p.kp[i] = int4 ? static_cast<uint8_t*>(const_cast<void*>(l.k_param)) : nullptr;
      p.vp[i] = int4 ? static_cast<uint8_t*>(const_cast<void*>(l.v_param)) : nullptr;
    }
    KB_LAUNCH("evict_move_kernel", launch_pdl(evict_move_kernel, dim3(ceil_div(max_moves, 8), n, batch), 256, 0, st, 1, p));
  }
  return 0;
}
}  // namespace kb200

extern "C" size_t kb200_evict_workspace_bytes(int batch, int n_rows, int budget) {
  if (batch <= 0 || n_rows <= 0 || budget <= 0) return 0;
  return (size_t)kb200::EvictWorkspace(batch, n_rows, budget).words * 4;
}

extern "C" int kb200_evict(const kb200_kv_layout* layers, int n_layers, const int32_t* seq_lens, const float* mass,
                           int64_t mass_stride, const int32_t* token_positions, int64_t pos_stride, int budget, int recent,
                           int sinks, int32_t* new_lens, float* mass_out, int32_t* pos_out, int64_t out_stride, void* workspace,
                           size_t workspace_bytes, int batch, int num_kv_heads, int n_rows, void* stream) {
  using namespace kb200;
  KB_ENTRY(mass, "evict: mass");
  KB_REQUIRE(layers && seq_lens && mass && new_lens && mass_out && pos_out, "evict: null pointer");
  KB_REQUIRE(n_layers >= 1 && batch >= 0 && batch <= 65535 && num_kv_heads > 0 && n_rows >= 0, "evict: bad sizes");
  KB_REQUIRE(budget >= 1 && budget <= (n_rows > 1 ? n_rows : 1) && recent >= 0 && sinks >= 0 && (int64_t)recent + sinks <= budget,
             "evict: a budget of %d rows of %d, %d first and %d last ones protected", budget, n_rows, sinks, recent);
  KB_REQUIRE(batch <= 1 || (mass_stride >= n_rows && (!token_positions || pos_stride >= n_rows)),
             "evict: rows of mass or token_positions overlap: %lld and %lld apart, %d long", (long long)mass_stride, (long long)pos_stride, n_rows);
  KB_REQUIRE(out_stride >= n_rows && mass_out != mass && pos_out != token_positions,
             "evict: outputs must hold %d rows and not be inputs", n_rows);
  if (check_layers(layers, n_layers) != 0) return -1;
  if (batch == 0) return 0;
  if (n_rows == 0) {
    KB_CUDA(cudaMemsetAsync(new_lens, 0, (size_t)batch * 4, (cudaStream_t)stream));
    return 0;
  }
  const EvictWorkspace at(batch, n_rows, budget);
  KB_REQUIRE(workspace && workspace_bytes >= (size_t)at.words * 4 && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
             "evict: a 16-byte aligned workspace of %lld bytes is required, got %zu", (long long)at.words * 4, workspace_bytes);
  int32_t* ws = static_cast<int32_t*>(workspace);
  float* keys = reinterpret_cast<float*>(ws);
  cudaStream_t st = (cudaStream_t)stream;
  // CTAs of a sequence: of 1024 rows at least, while there are SMs for them
  int ctas = 1;
  while (ctas < 8 && n_rows > ctas * 2048 && batch * ctas <= sm_count() / 2) ctas *= 2;
  KB_LAUNCH("evict_keys_kernel",
            launch_pdl(evict_keys_kernel, dim3(batch * ctas), kKeyThreads, 0, st, ctas,
                       EvictKeysParams{mass, mass_stride, seq_lens, token_positions, pos_stride, keys, at.keys_row, sinks, recent, budget, n_rows}));
  if (kb200_topk_select(keys, at.keys_row, n_rows, seq_lens, nullptr, budget, ws + at.keep, budget, ws + at.keep_count, batch, stream) != 0)
    return -1;
  int2* moves = reinterpret_cast<int2*>(ws + at.moves);
  KB_LAUNCH("evict_plan_kernel",
            launch_pdl(evict_plan_kernel, dim3(ceil_div(n_rows, 256), batch), 256, 0, st, 1,
                       EvictPlanParams{ws + at.keep, budget, ws + at.keep_count, mass, mass_stride, token_positions, pos_stride, moves,
                                       ws + at.move_count, new_lens, mass_out, pos_out, out_stride, n_rows}));
  const int max_moves = n_rows - budget < budget ? n_rows - budget : budget;
  return max_moves > 0 ? move_rows(layers, n_layers, moves, budget, ws + at.move_count, max_moves, batch, num_kv_heads, st) : 0;
}
