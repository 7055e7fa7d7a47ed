// Paged decode attention over a 4-bit KV cache (KB200_INT4), sparse (reuse layers) and dense (anchor layers).
//
// A row of 128 values is four groups of 32 codes c in 0..15 that stand for s c + z, with s and z in fp16 per group; the
// order of the codes in a row is written beside kb200_kv_layout.  Same division of the work as in decode.cu: a CTA owns one
// (sequence, KV head, split), and its partial results meet in merge_warps and decode_combine_kernel.
//
// One warp per key: a lane holds four values of the row (16 bits of codes).
#include "decode.cuh"

namespace kb200 {

constexpr int kWarps4 = 8;

template <bool DENSE, bool HAS_V, bool BF16>
__global__ void __launch_bounds__(kWarps4 * 32) decode_attn4_kernel(const DecodeParams p) {
  pdl_wait();
  constexpr uint32_t FULL = 0xFFFFFFFFu;
  __shared__ float sm_m[kWarps4 * kHg], sm_l[kWarps4 * kHg], sm_o[HAS_V ? kWarps4 * kHg * kD : 1];
  const int split = blockIdx.x, g = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
  const int nst = (n + 15) / 16, per = (nst + p.num_splits - 1) / p.num_splits;
  const int begin = min(split * per * 16, n), end = min(begin + per * 16, n);

  // the values of this lane: nibbles 4 lane .. 4 lane + 3 of a row
  const int k_group = (lane & 7) >> 1, k_d = 32 * k_group + 8 * (lane >> 3) + 4 * (lane & 1);
  const int v_group = lane & 3, v_d = 32 * v_group + 4 * (lane >> 2);
  float q[kHg][4];
#pragma unroll
  for (int h = 0; h < kHg; ++h) {
    const __half* qp = p.q + b * p.q_stride_b + (int64_t)(g * kHg + h) * p.q_stride_h + k_d;
#pragma unroll
    for (int e = 0; e < 4; ++e) q[h][e] = BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(qp)[e]) : __half2float(qp[e]);
  }
  const uint8_t* k8 = reinterpret_cast<const uint8_t*>(p.k) + (int64_t)b * p.kv_stride_batch + (int64_t)g * p.kv_stride_head;
  const uint8_t* v8 = reinterpret_cast<const uint8_t*>(p.v) + (int64_t)b * p.kv_stride_batch + (int64_t)g * p.kv_stride_head;
  const int64_t pa_base = (int64_t)b * p.pa_stride_batch + (int64_t)g * p.pa_stride_head;
  float m[kHg], l[kHg], o[kHg][4];
#pragma unroll
  for (int h = 0; h < kHg; ++h) {
    m[h] = -INFINITY;
    l[h] = o[h][0] = o[h][1] = o[h][2] = o[h][3] = 0.f;
  }
  for (int j = begin + warp; j < end; j += kWarps4) {
    const int pos = DENSE ? j : idx_row[j];
    const int lp = pos >> p.page_shift, slot = pos & p.page_mask;
    const int64_t page = p.block_table ? p.block_table[(int64_t)b * p.block_table_stride + lp] : lp;
    const int64_t at = page * p.kv_stride_page + slot * p.kv_stride_token;
    const int64_t pa = pa_base + page * p.pa_stride_page + slot * p.pa_stride_token;
    const uint32_t kc = reinterpret_cast<const uint16_t*>(k8 + at)[lane];
    const float ks = __half2float(p.k_param[pa + k_group]), kz = __half2float(p.k_param[pa + 4 + k_group]);
    float x[kHg];
#pragma unroll
    for (int h = 0; h < kHg; ++h) {
      x[h] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[h] += q[h][e] * (ks * (float)((kc >> (4 * e)) & 15) + kz);
#pragma unroll
      for (int sh = 16; sh > 0; sh >>= 1) x[h] += __shfl_xor_sync(FULL, x[h], sh);
      x[h] *= p.scale2;
    }
    if (DENSE && lane < kHg) {
      float mine = x[0];
#pragma unroll
      for (int h = 1; h < kHg; ++h) mine = lane == h ? x[h] : mine;
      p.logits[((int64_t)b * p.H + g * kHg + lane) * p.logit_stride + j] = mine;
    }
    float v[4];
    if (HAS_V) {
      const uint32_t vc = reinterpret_cast<const uint16_t*>(v8 + at)[lane];
      const float vs = __half2float(p.v_param[pa + v_group]), vz = __half2float(p.v_param[pa + 4 + v_group]);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = vs * (float)((vc >> (4 * e)) & 15) + vz;
    }
#pragma unroll
    for (int h = 0; h < kHg; ++h) {
      const float m_new = fmaxf(m[h], x[h]);
      const float alpha = exp2f(m[h] - m_new), w = exp2f(x[h] - m_new);
      m[h] = m_new;
      l[h] = l[h] * alpha + w;
      if (HAS_V) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[h][e] = o[h][e] * alpha + w * v[e];
      }
    }
  }
  pdl_trigger();
#pragma unroll
  for (int h = 0; h < kHg; ++h) {
    if (lane == 0) { sm_m[warp * kHg + h] = m[h]; sm_l[warp * kHg + h] = l[h]; }
    if (HAS_V) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sm_o[(warp * kHg + h) * kD + v_d + e] = o[h][e];
    }
  }
  __syncthreads();
  merge_warps<HAS_V, BF16>(p, sm_m, sm_l, sm_o, kWarps4, b, g, split);
}

int init_decode4() { return 0; }

cudaError_t launch_attn4(const DecodeParams& p, bool dense, bool has_v, dim3 grid, cudaStream_t st) {
  auto* kernel = !dense ? (p.bf16 ? decode_attn4_kernel<false, true, true> : decode_attn4_kernel<false, true, false>)
                 : !has_v ? (p.bf16 ? decode_attn4_kernel<true, false, true> : decode_attn4_kernel<true, false, false>)
                 : p.bf16 ? decode_attn4_kernel<true, true, true> : decode_attn4_kernel<true, true, false>;
  return launch_pdl(kernel, grid, kWarps4 * 32, 0, st, 1, p);
}

}  // namespace kb200
