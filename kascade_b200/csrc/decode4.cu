// Paged decode attention over a 4-bit KV cache (KB200_INT4), sparse (reuse layers) and dense (anchor layers).
//
// A row of 128 values is four groups of 32 codes c in 0..15 that stand for s c + z, with s and z in fp16 per group; the
// order of the codes in a row is written beside kb200_kv_layout.  Same division of the work as in decode.cu: a CTA owns one
// (sequence, KV head, split), every warp streams steps of 32 keys through a private cp.async ring, and partial results meet in
// merge_warps and decode_combine_kernel.
//
// At 160 bytes a key the copies leave a warp scheduler some 230 issue slots per eight keys, so the rows are never turned into
// fp16 values.  A code in the low bits of an fp16 word IS a number: the subnormal c 2^-24, or 16 c 2^-24 four bits further
// up, and the tensor core takes subnormals as they are.  One AND therefore makes a pair of matrix operands from a word of
// codes (two, after a shift), and scales and zeros are applied where they are few:
//   * S = K Q^T, keys as rows:  S = sum_g s_g (sum_{d in g} c_d q_d) + sum_g z_g (sum_{d in g} q_d).  Two products of 16 d for each
//     group, whose sums are scaled by the key's s_g in fp32; the zeros are one more product, of the keys' parameters with the
//     queries' sums over the groups (as two fp16 terms, exact to 2^-22).
//   * O^T = V^T P^T, values as rows:  sum_k (p_k s_gk) c_dk  with the scale on the probabilities, which are one row per head,
//     not on the 128 values, and sum_k p_k z_gk as one product with the transposed parameters.
// The orders of the codes in K and V rows are those in which a lane needs them: 16 bytes of a K row, 8 of a V row.
// What bounds it: dense passes and rows in order, HBM (5.5-5.6 TB/s at 37 x 16384 and 64 x 32768 keys; 128 us of 144 for the
// former with the cache in L2, with 59 % of the issue slots and 52 % of the integer pipe busy); reuse layers, lines: DRAM hands
// out 128 bytes at a time, so random rows of 64 + 64 + 32 bytes move 304 bytes per key (64 x 3244 rows: 95 us, 5.3 TB/s of DRAM
// traffic).
// Queries are brought to a largest element of 64..128 per head by a power of two, so that bf16 ones fit fp16 exactly.
#include "decode.cuh"

namespace kb200 {

constexpr int kWarps4 = 16;                                // warps of a full-size CTA (one per SM); half-size CTAs run two per SM
constexpr int kKeys4 = 32;                                 // keys of a step, one per lane while they are copied
constexpr int kCodes4 = kKeys4 * kD / 2;                   // bytes of the codes of a step's K or V rows
constexpr int kHalf4 = kCodes4 + kKeys4 * 16;              // ... with their parameters
constexpr int kCodeOne = 1 << 24;                          // 1 / (the value of code 1 as an fp16 subnormal)
// A row's reference point for its exponentials lies kBase4 below the largest logit (in units of log2) when it is set, and moves only
// when a logit exceeds it by more than kTop4: the maximum over the lanes, the factors and the rescaling of O are needed in a
// few steps per list only.  So the probabilities p are at most 2^13 and the largest of a warp is 2^11 at least, and fp16 holds
// all that are more than 2^-25 of the largest with all of its bits.
constexpr float kBase4 = 11.f, kTop4 = 13.f;
// Scales get a power of two of their own, per warp and group: 2^up brings the largest scale so far to [2, 4), so that p s 2^up stays
// below 2^15 and, like p, keeps its bits down to 2^-26 of the largest, whatever the size of V.  It moves as the reference does.
// (Without it p s falls below 2^-14, where fp16 has steps of 2^-24, wherever V is small or one key dominates: for 8192 keys with
// one 9 above the others and V of a standard deviation of 0.03 outputs were off by 17 %.)  Scales below 2^-15 are taken
// times 2^15, the largest power of two in fp16.  It takes 1 % of a dense pass of K and V and of a reuse layer (16 ragged sequences of
// up to 32768 keys 147.4 -> 149.3 us, 64 x 3244 rows 117.2 -> 118.7, whole layers, L2 flushed).
constexpr int kMaxUp4 = 15;
constexpr float kUnbase4 = 1.f / 2048.f;                   // 2^-kBase4: the results are relative to the largest logit again
// The tensor core rounds its sums towards zero: by about 2^-24 of the accumulator per product, always the same way.  The codes' mean
// is 7.5, so their share of O grows with the list while O itself, with the zeros' share taken off, does not: after 512 products that
// was 0.4 % of O for 131072 keys.  (And it aligns products by their operands' exponent fields, so a subnormal loses what it lies below
// 2^-14; V's codes are shifted two bits up for that.)  So every kFlush4 steps what the accumulators of a group have in common (one
// of them) is taken off all of them and added up apart, rounded to nearest, in a few words per lane of shared memory.  Error of
// fp16 outputs against 64 bits, 131072 keys in 1 / 18 splits: 4.0e-3 / 5.3e-4 without, 6e-4 unshifted, 3.0e-4 / 2.8e-4 as it is
// (2.9e-4 is what the rounding of probabilities and outputs to fp16 makes); every 8 steps 3.3e-4, every 16 4.6e-4.  It takes 1-2 %
// of a dense pass.
constexpr int kFlush4 = 4;
constexpr int kTracks4 = 10;                               // per lane: four groups and the zeros, two heads each
constexpr int kTrackBytes4 = kTracks4 * 32 * 4;            // per warp
__host__ __device__ constexpr int stages4(bool has_v) { return has_v ? 2 : 4; }
__host__ __device__ constexpr int stage_bytes4(bool has_v) { return has_v ? 2 * kHalf4 : kHalf4; }
__host__ __device__ constexpr int warp_bytes4(bool has_v) { return stages4(has_v) * stage_bytes4(has_v) + (has_v ? kTrackBytes4 : 0); }

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void ldmatrix_x2(uint32_t& a, uint32_t& b, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];\n" : "=r"(a), "=r"(b) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x2_trans(uint32_t& a, uint32_t& b, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];\n" : "=r"(a), "=r"(b) : "r"(addr));
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(r.x), "=r"(r.y) : "r"(addr));
  return r;
}
__device__ __forceinline__ float2 half2_floats(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t fma_half2(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                            *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// The sequence of rank r by length, the longest first (equal lengths by position), found by all threads of the CTA; `lens` is n + 1
// words of shared memory, free again when it returns.  A long sequence whose CTAs start last runs alone at the end.  us of a dense pass
// with sequences as they come / the longest first, in the best number of splits of either: 8 of up to 32768 keys 60.7 / 62.4, 16 109
// / 104, 64 434 / 376, 24 and 32 and 48 of up to 16384 93.5 / 88.4, 114 / 102 and 167 / 143, 64 of up to 8192 108 / 99.5.  Sequences
// of one length pay for it: 64 x 4096 96.0 / 97.5, 64 x 16384 332.8 / 333.3; 200 x 2048, which are not ranked, 129 / 147.
constexpr int kRankMax4 = 64;
__device__ __forceinline__ int longest_first4(int r, int n, const int32_t* seq_lens, int* lens) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) lens[i] = seq_lens[i];
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int mine = lens[i];
    int before = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) before += lens[j] > mine || (lens[j] == mine && j < i);
    if (before == r) lens[n] = i;
  }
  __syncthreads();
  const int b = lens[n];
  __syncthreads();
  return b;
}

template <bool DENSE, bool HAS_V, bool BF16>
__global__ void __launch_bounds__(kWarps4 * 32, 1) decode_attn4_kernel(const DecodeParams p) {
  pdl_wait();
  constexpr uint32_t FULL = 0xFFFFFFFFu;
  constexpr int kStages = stages4(HAS_V), kStage = stage_bytes4(HAS_V);
  const int WARPS = blockDim.x >> 5;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int split = blockIdx.x, g = blockIdx.y;
  const int b = DENSE && p.by_length ? longest_first4(blockIdx.z, gridDim.z, p.seq_lens, reinterpret_cast<int*>(smem))
                                     : (int)blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grp = lane >> 2, quad = lane & 3;

  // ---- this CTA's slice of the key list, in steps of 32 keys --------------------------------------
  int n;
  const int32_t* idx_row = nullptr;
  if (DENSE) {
    n = p.seq_lens[b];
  } else {
    const int src_g = p.head_map ? p.head_map[g] : g;
    n = min(p.count ? p.count[b * p.G + src_g] : p.k_max, p.k_max);
    idx_row = p.idx + b * p.idx_stride_b + src_g * p.idx_stride_g;
  }
  n = max(n, 0);
  const int nst = (n + kKeys4 - 1) / kKeys4, per = (nst + p.num_splits - 1) / p.num_splits;
  const int st_begin = min(split * per, nst), st_end = min(st_begin + per, nst);
  const int my_count = (st_end - st_begin - warp + WARPS - 1) / WARPS;                 // may be <= 0

  // ---- queries: B operand Q^T[d][head], columns 0-3 = heads 0-3, 4-7 = the same again ---------------
  // k-step (group e, half f): k = 2 quad, 2 quad + 1 are d = 32 e + 8 quad + {2f, 2f + 4}, k + 8 the d one further, whose codes
  // lie four bits further up: times 4 here, a quarter there
  uint32_t qb[4][2][2], zb0, zb1;
  float c_head[2];                                         // scale * log2 e * 2^(exponent of the head's queries), columns 2 quad, + 1
  {
    const __half* qp = p.q + b * p.q_stride_b + (int64_t)(g * kHg + (grp & 3)) * p.q_stride_h;
    float q[4][8], top = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(qp + 32 * e + 8 * quad + 2 * i);
        const float2 f = BF16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w)) : half2_floats(w);
        q[e][2 * i] = f.x;
        q[e][2 * i + 1] = f.y;
        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
    top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
    const int up = 6 - max((int)(__float_as_uint(top) >> 23) - 127, -90);   // exponent of the factor: -121 .. 96
    const float factor = __uint_as_float((uint32_t)(up + 127) << 23);
    const float unit = p.scale2 * __uint_as_float((uint32_t)(127 - up) << 23);
    c_head[0] = __shfl_sync(FULL, unit, (quad & 1) * 8);
    c_head[1] = __shfl_sync(FULL, unit, (quad & 1) * 8 + 4);
    float sum[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sum[e] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        q[e][i] = __half2float(__float2half_rn(q[e][i] * factor));
        sum[e] += q[e][i];
      }
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        qb[e][f][0] = pack_half2<false>(q[e][2 * f] * 4.f, q[e][2 * f + 4] * 4.f);
        qb[e][f][1] = pack_half2<false>(q[e][2 * f + 1] * 0.25f, q[e][2 * f + 5] * 0.25f);
      }
      sum[e] += __shfl_xor_sync(FULL, sum[e], 1);
      sum[e] += __shfl_xor_sync(FULL, sum[e], 2);
    }
    // zeros: k = 4 + e of the parameters is z_e; the high parts of the sums below, the rests in k + 8
    const float s0 = quad == 2 ? sum[0] : sum[2], s1 = quad == 2 ? sum[1] : sum[3];
    zb0 = quad < 2 ? 0u : pack_half2<false>(s0, s1);
    const float2 high = half2_floats(zb0);
    zb1 = quad < 2 ? 0u : pack_half2<false>(s0 - high.x, s1 - high.y);
  }

  const uint8_t* k_base = reinterpret_cast<const uint8_t*>(p.k) + (int64_t)b * p.kv_stride_batch + (int64_t)g * p.kv_stride_head;
  const uint8_t* v_base = reinterpret_cast<const uint8_t*>(p.v) + (int64_t)b * p.kv_stride_batch + (int64_t)g * p.kv_stride_head;
  const __half* kp_base = p.k_param + (int64_t)b * p.pa_stride_batch + (int64_t)g * p.pa_stride_head;
  const __half* vp_base = p.v_param + (int64_t)b * p.pa_stride_batch + (int64_t)g * p.pa_stride_head;
  const int32_t* table = p.block_table ? p.block_table + (int64_t)b * p.block_table_stride : nullptr;
  const uint32_t ring = smem_u32(smem) + warp * (kStages * kStage);

  // Codes in shared memory: two rows to a line of 128 bytes, the 16-byte pieces of line i exchanged by XOR with 2 i, so that
  // the copies, the reads of K (eight pieces of a line at once) and of V (two pieces of four lines) use all banks.
  // A lane copies piece quad of row grp (+ 8 i) and later reads the same piece of K.
  const uint32_t k_at = (lane >> 3) * 128 + (((lane & 7) ^ ((lane >> 3) * 2)) << 4);
  const uint32_t v_at = quad * 128 + (((grp >> 1) ^ (quad * 2)) << 4) + (grp & 1) * 8;   // row 2 quad, bytes 8 grp ..; the next row: ^ 64

  auto load_pos = [&](int j) -> int {                      // position of key `lane` of step j of this warp
    if (j >= my_count) return 0;
    const int s = min((st_begin + warp + j * WARPS) * kKeys4 + lane, n - 1);
    return DENSE ? s : idx_row[s];
  };
  auto load_page = [&](int pos) -> int {
    const int lp = pos >> p.page_shift;
    return table ? table[lp] : lp;
  };
  auto issue = [&](int j, int pos, int page) {
    if (j < my_count) {
      const int slot = pos & p.page_mask;
      const int64_t off = (int64_t)page * p.kv_stride_page + (int64_t)slot * p.kv_stride_token;
      const int64_t par = (int64_t)page * p.pa_stride_page + (int64_t)slot * p.pa_stride_token;
      const uint32_t dst = ring + (j % kStages) * kStage;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t row = __shfl_sync(FULL, off, i * 8 + grp) + quad * 16;
        cp_async16(dst + i * 512 + k_at, k_base + row);
        if (HAS_V) cp_async16(dst + kHalf4 + i * 512 + k_at, v_base + row);
      }
      cp_async16(dst + kCodes4 + lane * 16, kp_base + par);
      if (HAS_V) cp_async16(dst + kHalf4 + kCodes4 + lane * 16, vp_base + par);
    }
    cp_async_commit();
  };

  int pos_a, page_a, pos_b;
  {
    int pos[kStages], page[kStages];
#pragma unroll
    for (int i = 0; i < kStages; ++i) pos[i] = load_pos(i);
#pragma unroll
    for (int i = 0; i < kStages; ++i) page[i] = load_page(pos[i]);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i, pos[i], page[i]);
    pos_a = pos[kStages - 1];
    page_a = page[kStages - 1];
    pos_b = load_pos(kStages);
  }

  // o_acc[e][f]: values d = 32 e + 4 grp + 2 f (rows 0-7) and + 1, times 16 (rows 8-15), of heads 2 quad, 2 quad + 1; o_zero: row
  // 4 + e is the zeros' share of group e
  float o_acc[4][2][4], o_zero[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    o_zero[e] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) o_acc[e][0][i] = o_acc[e][1][i] = 0.f;
  }
  float m_run[2] = {-INFINITY, -INFINITY}, l_part[2] = {0.f, 0.f};
  int up = grp < 4 ? kMaxUp4 : 0;                                // lane (e, quad): the power of two of group e's scales (the zeros have none)
  float* track = reinterpret_cast<float*>(smem + WARPS * (kStages * kStage) + warp * kTrackBytes4) + lane;   // [10], 32 apart
  if (HAS_V) {
#pragma unroll
    for (int i = 0; i < kTracks4; ++i) track[i * 32] = 0.f;
  }
  auto flush = [&] {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float mean = o_acc[e][0][r];
        track[(e * 2 + r) * 32] += mean;
        o_acc[e][0][r] = 0.f;
        o_acc[e][1][r] -= mean;
        o_acc[e][0][2 + r] = fmaf(-16.f, mean, o_acc[e][0][2 + r]);
        o_acc[e][1][2 + r] = fmaf(-16.f, mean, o_acc[e][1][2 + r]);
      }
      track[(8 + r) * 32] += o_zero[r];
      o_zero[r] = 0.f;
    }
  };

  // p s in fp16 for columns 0-3, and for columns 4-7 (the same heads) what its rounding left (exactly where p s, which goes up to 2^15,
  // is 2^-3 or more): the products with the codes, whose mean is far from zero, would carry the rounding of p s twice as far as
  // that of p.  bf16 outputs are rounded ten times as coarsely and do without.
  const uint32_t rest = grp < kHg ? 0u : 0xFFFFFFFFu;
  auto scaled = [&](uint32_t pb, uint32_t s) -> uint32_t {
    const uint32_t ps = mul_half2(pb, s);
    return BF16 ? ps : fma_half2(pb, s, (ps ^ 0x80008000u) & rest);
  };

  for (int j = 0; j < my_count; ++j) {
    __syncwarp();                      // every lane is done with the buffer about to be refilled
    issue(j + kStages - 1, pos_a, page_a);
    pos_a = pos_b;
    page_a = load_page(pos_a);
    pos_b = load_pos(j + kStages + 1);
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const uint32_t buf = ring + (j % kStages) * kStage;
    const int key0 = (st_begin + warp + j * WARPS) * kKeys4;

    // ---- logits: x[i] of keys 16 i + grp and + 8, heads 2 quad, 2 quad + 1 -------------------------------
    float x[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t wa[4], wb[4];                                 // group e's eight codes of keys grp and grp + 8
      lds128(wa[0], wa[1], wa[2], wa[3], buf + i * 1024 + k_at);
      lds128(wb[0], wb[1], wb[2], wb[3], buf + i * 1024 + 512 + k_at);
      const uint32_t par = buf + kCodes4 + i * 256;
      uint32_t za, zc;
      ldmatrix_x2(za, zc, par + (lane & 15) * 16);
      float zero[4] = {0.f, 0.f, 0.f, 0.f}, t[4] = {0.f, 0.f, 0.f, 0.f};
      mma16816<false>(zero, za, zc, za, zc, zb0, zb1);
      const uint2 sa = lds64(par + grp * 16), sb = lds64(par + grp * 16 + 128);
      const float2 sa01 = half2_floats(sa.x), sa23 = half2_floats(sa.y), sb01 = half2_floats(sb.x), sb23 = half2_floats(sb.y);
      const float fa[4] = {sa01.x, sa01.y, sa23.x, sa23.y}, fb[4] = {sb01.x, sb01.y, sb23.x, sb23.y};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        mma16816<false>(s, wa[e] & 0x000F000Fu, wb[e] & 0x000F000Fu, wa[e] & 0x00F000F0u, wb[e] & 0x00F000F0u, qb[e][0][0], qb[e][0][1]);
        const uint32_t ha = wa[e] >> 8, hb = wb[e] >> 8;
        mma16816<false>(s, ha & 0x000F000Fu, hb & 0x000F000Fu, ha & 0x00F000F0u, hb & 0x00F000F0u, qb[e][1][0], qb[e][1][1]);
        t[0] += fa[e] * s[0];
        t[1] += fa[e] * s[1];
        t[2] += fb[e] * s[2];
        t[3] += fb[e] * s[3];
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) x[i][r] = fmaf(t[r], (float)(kCodeOne / 4), zero[r]) * c_head[r & 1];
    }
    if (key0 + kKeys4 > n) {                                 // the list ends inside this step
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (key0 + 16 * i + grp >= n) x[i][0] = x[i][1] = -INFINITY;
        if (key0 + 16 * i + grp + 8 >= n) x[i][2] = x[i][3] = -INFINITY;
      }
    }
    if (DENSE) {
      // columns 4-7 are the same heads again: the lanes of quads 0, 1 write the first 16 keys, the others the last
      const int half = quad >> 1;
      float* lp = p.logits + ((int64_t)b * p.H + g * kHg + (quad & 1) * 2) * p.logit_stride + key0 + 16 * half + grp;
      const int keys = n - (key0 + 16 * half + grp);
      if (keys > 0) { lp[0] = half ? x[1][0] : x[0][0]; lp[p.logit_stride] = half ? x[1][1] : x[0][1]; }
      if (keys > 8) { lp[8] = half ? x[1][2] : x[0][2]; lp[p.logit_stride + 8] = half ? x[1][3] : x[0][3]; }
    }
    // ---- exponentials against the reference of either head ---------------------------------------------
    float t0 = fmaxf(fmaxf(x[0][0], x[0][2]), fmaxf(x[1][0], x[1][2])), t1 = fmaxf(fmaxf(x[0][1], x[0][3]), fmaxf(x[1][1], x[1][3]));
    uint32_t z[2][2];                                        // lane (r, quad): parameter r of keys 2 quad, 2 quad + 1 / + 8 of either 16
    __half2 top = __half2half2(__ushort_as_half(0));
    if (HAS_V) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ldmatrix_x2_trans(z[i][0], z[i][1], buf + kHalf4 + kCodes4 + i * 256 + (lane & 15) * 16);
        top = __hmax2(top, __hmax2(__habs2(*reinterpret_cast<__half2*>(&z[i][0])), __habs2(*reinterpret_cast<__half2*>(&z[i][1]))));
      }
    }
    // (a scale of 2^(2 - up) or more; the first step moves in any case: it has a valid key)
    const bool grown = HAS_V && grp < 4 && !__hblt2(top, __half2half2(__float2half_rn(__uint_as_float((uint32_t)(129 - up) << 23))));
    if (__any_sync(FULL, grown || t0 > m_run[0] + kTop4 || t1 > m_run[1] + kTop4)) {
#pragma unroll
      for (int sh = 4; sh <= 16; sh <<= 1) {
        t0 = fmaxf(t0, __shfl_xor_sync(FULL, t0, sh));
        t1 = fmaxf(t1, __shfl_xor_sync(FULL, t1, sh));
      }
      const float m0 = t0 > m_run[0] + kTop4 ? t0 - kBase4 : m_run[0], m1 = t1 > m_run[1] + kTop4 ? t1 - kBase4 : m_run[1];
      const float alpha0 = ex2(m_run[0] - m0), alpha1 = ex2(m_run[1] - m1);
      m_run[0] = m0;
      m_run[1] = m1;
      l_part[0] *= alpha0;
      l_part[1] *= alpha1;
      if (HAS_V) {
        float s_top = fmaxf(__low2float(top), __high2float(top));
        s_top = fmaxf(s_top, __shfl_xor_sync(FULL, s_top, 1));
        s_top = fmaxf(s_top, __shfl_xor_sync(FULL, s_top, 2));
        const int to = grp < 4 ? max(min(up, 128 - (int)(__float_as_uint(s_top) >> 23)), -14) : up;
        const float ratio = __uint_as_float((uint32_t)(127 + to - up) << 23);
        up = to;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float r = __shfl_sync(FULL, ratio, e * 4 + quad), r0 = alpha0 * r, r1 = alpha1 * r;
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            o_acc[e][f][0] *= r0; o_acc[e][f][1] *= r1; o_acc[e][f][2] *= r0; o_acc[e][f][3] *= r1;
          }
          track[(2 * e) * 32] *= r0;
          track[(2 * e + 1) * 32] *= r1;
        }
        o_zero[0] *= alpha0; o_zero[1] *= alpha1;
        track[8 * 32] *= alpha0;
        track[9 * 32] *= alpha1;
      }
    }
    float w[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) w[i][r] = ex2(x[i][r] - m_run[r & 1]);
    }
    l_part[0] += (w[0][0] + w[0][2]) + (w[1][0] + w[1][2]);
    l_part[1] += (w[0][1] + w[0][3]) + (w[1][1] + w[1][3]);
    if (HAS_V) {
      // ---- O^T += V^T P^T -------------------------------------------------------------------------------
      const __half up_h = __float2half_rn(__uint_as_float((uint32_t)(127 + up) << 23));
      const __half2 up2_h = __half2half2(up_h);
      const uint32_t up2 = *reinterpret_cast<const uint32_t*>(&up2_h);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // B operand P^T[key][head]: column = head grp, rows = keys 2 quad, 2 quad + 1 (pb0) and + 8 (pb1)
        const uint32_t pb0 = movmatrix_trans(pack_half2<false>(w[i][0], w[i][1]));
        const uint32_t pb1 = movmatrix_trans(pack_half2<false>(w[i][2], w[i][3]));
        const uint32_t z0 = mul_half2(z[i][0], up2), z1 = mul_half2(z[i][1], up2);
        mma16816<false>(o_zero, z0, 0u, z1, 0u, pb0, pb1);
        const uint32_t v = buf + kHalf4 + i * 1024 + v_at;
        const uint2 ka = lds64(v), kb = lds64(v ^ 64u), kc = lds64(v + 512), kd = lds64((v + 512) ^ 64u);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t sel = (e & 1) ? 0x7632 : 0x5410;
          const uint32_t lo = __byte_perm(e < 2 ? ka.x : ka.y, e < 2 ? kb.x : kb.y, sel);      // keys 2 quad, 2 quad + 1
          const uint32_t hi = __byte_perm(e < 2 ? kc.x : kc.y, e < 2 ? kd.x : kd.y, sel);      // ... + 8
          const uint32_t sb0 = scaled(pb0, __shfl_sync(FULL, z0, e * 4 + quad));
          const uint32_t sb1 = scaled(pb1, __shfl_sync(FULL, z1, e * 4 + quad));
          const uint32_t lo2 = lo << 2, hi2 = hi << 2, lo6 = lo >> 6, hi6 = hi >> 6;
          mma16816<false>(o_acc[e][0], lo2 & 0x003C003Cu, lo2 & 0x03C003C0u, hi2 & 0x003C003Cu, hi2 & 0x03C003C0u, sb0, sb1);
          mma16816<false>(o_acc[e][1], lo6 & 0x003C003Cu, lo6 & 0x03C003C0u, hi6 & 0x003C003Cu, hi6 & 0x03C003C0u, sb0, sb1);
        }
      }
      if ((j & (kFlush4 - 1)) == kFlush4 - 1) flush();
    }
  }
  cp_async_wait<0>();
  if (HAS_V) {                         // what was taken off comes back, rounded to nearest like every sum of it
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float mean = track[(e * 2 + r) * 32];
        o_acc[e][0][r] += mean;
        o_acc[e][1][r] += mean;
        o_acc[e][0][2 + r] = fmaf(16.f, mean, o_acc[e][0][2 + r]);
        o_acc[e][1][2 + r] = fmaf(16.f, mean, o_acc[e][1][2 + r]);
      }
      o_zero[r] += track[(8 + r) * 32];
    }
  }
  __syncthreads();
  pdl_trigger();                       // only the merge is left: most SMs have room by now

#pragma unroll
  for (int sh = 4; sh <= 16; sh <<= 1) {
    l_part[0] += __shfl_xor_sync(FULL, l_part[0], sh);
    l_part[1] += __shfl_xor_sync(FULL, l_part[1], sh);
  }
  float* sm_m = reinterpret_cast<float*>(smem);                  // [warps][4]
  float* sm_l = sm_m + WARPS * kHg;                              // [warps][4]
  float* sm_o = sm_l + WARPS * kHg;                              // [warps][4][128]
  float zero[4][2], unit[4];                                     // what group e's sums of p s c are multiplied by in the end
  if (HAS_V && !BF16) {                                          // the rests, columns 4-7, to their heads
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o_acc[e][0][i] += __shfl_down_sync(FULL, o_acc[e][0][i], 2);
        o_acc[e][1][i] += __shfl_down_sync(FULL, o_acc[e][1][i], 2);
      }
    }
  }
  if (HAS_V) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      zero[e][0] = __shfl_sync(FULL, o_zero[0], (4 + e) * 4 + quad) * kUnbase4;
      zero[e][1] = __shfl_sync(FULL, o_zero[1], (4 + e) * 4 + quad) * kUnbase4;
      unit[e] = __uint_as_float((uint32_t)(127 + 22 - (int)kBase4 - __shfl_sync(FULL, up, e * 4 + quad)) << 23);
    }
  }
  if (quad < 2) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int h = quad * 2 + r;
      if (grp == 0) { sm_m[warp * kHg + h] = m_run[r] + kBase4; sm_l[warp * kHg + h] = l_part[r] * kUnbase4; }
      if (HAS_V) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float4 o;
          o.x = fmaf(o_acc[e][0][r], unit[e], zero[e][r]);
          o.y = fmaf(o_acc[e][0][2 + r], unit[e] / 16, zero[e][r]);
          o.z = fmaf(o_acc[e][1][r], unit[e], zero[e][r]);
          o.w = fmaf(o_acc[e][1][2 + r], unit[e] / 16, zero[e][r]);
          *reinterpret_cast<float4*>(sm_o + (warp * kHg + h) * kD + 32 * e + 4 * grp) = o;
        }
      }
    }
  }
  __syncthreads();
  merge_warps<HAS_V, BF16>(p, sm_m, sm_l, sm_o, WARPS, b, g, split);
}

template <bool DENSE, bool HAS_V>
static int init_one() {
  const int bytes = kWarps4 * warp_bytes4(HAS_V);
  KB_CUDA(cudaFuncSetAttribute(decode_attn4_kernel<DENSE, HAS_V, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  KB_CUDA(cudaFuncSetAttribute(decode_attn4_kernel<DENSE, HAS_V, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return 0;
}

int init_decode4() { return init_one<false, true>() || init_one<true, true>() || init_one<true, false>() ? -1 : 0; }

// CTAs of 16 warps, one per SM, while the grid is small; of 8, two per SM, from 1.5 CTAs per SM on, as in decode.cu; of 4, four per
// SM, from 6 on: there one CTA's start (lengths -> index -> block table -> rows) and merge are hidden behind three others.  us with 8 /
// 4 warps: reuse of 128 x 1606 rows 97.5 / 93.9, 256 x 787 102.7 / 94.2; dense passes of 256 x 2048 179 / 160, 16 of 5213..32768 rows in 7
// splits 115 / 111; but 64 x 3244 rows, 3.5 CTAs per SM, 93 / 102.
template <bool DENSE, bool HAS_V>
static cudaError_t launch(DecodeParams p, dim3 grid, cudaStream_t st) {
  const long long total = (long long)grid.x * grid.y * grid.z, sms = sm_count();
  const int warps = total >= 6 * sms ? kWarps4 / 4 : total * 2 >= 3 * sms ? kWarps4 / 2 : kWarps4;
  p.by_length = DENSE && grid.z > 1 && grid.z <= kRankMax4 && total > 2 * sms;      // more CTAs than start at once
  const size_t smem = (size_t)warps * warp_bytes4(HAS_V);
  return launch_pdl(p.bf16 ? decode_attn4_kernel<DENSE, HAS_V, true> : decode_attn4_kernel<DENSE, HAS_V, false>, grid, warps * 32, smem,
                    st, 1, p);
}

cudaError_t launch_attn4(const DecodeParams& p, bool dense, bool has_v, dim3 grid, cudaStream_t st) {
  return !dense ? launch<false, true>(p, grid, st) : has_v ? launch<true, true>(p, grid, st) : launch<true, false>(p, grid, st);
}

}  // namespace kb200
