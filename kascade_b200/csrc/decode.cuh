// What the decode kernels over 16-bit, FP8 and 4-bit caches share: their parameters, MMA helpers and the merge of a CTA's warps.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace kb200 {

struct DecodeParams {
  const __half* q;
  int64_t q_stride_b, q_stride_h;
  const __half* k;
  const __half* v;
  int64_t kv_stride_batch, kv_stride_page, kv_stride_token, kv_stride_head;
  const int32_t* block_table;
  int32_t block_table_stride;
  int32_t page_shift, page_mask;
  const int32_t* idx;            // sparse: index rows
  int64_t idx_stride_b, idx_stride_g;
  const int32_t* count;          // sparse: [B,G] valid entries (or NULL)
  int32_t k_max;
  const int32_t* head_map;       // sparse: [G] or NULL
  const int32_t* seq_lens;       // dense: [B]
  float scale2;                  // softmax_scale * log2(e)
  float* logits;                 // dense: [B,H,logit_stride]
  int64_t logit_stride;
  __half* out;                   // [B,H,D] (written here only when num_splits == 1)
  float* lse2;                   // [B,H]
  float* ws_m;                   // [B,H,S]
  float* ws_l;                   // [B,H,S]
  float* ws_o;                   // [B,H,S,D]
  int32_t H, G, num_splits;
  int32_t by_length;             // the longest sequences' CTAs come first (see longest_first)
  int32_t bf16;                  // host side: cache, q and the output are bf16, not fp16
  // FP8 (e4m3) cache: one fp32 scale per (page, KV head) for K and for V; q and the output are fp16
  int32_t fp8;
  const float* k_scale;
  const float* v_scale;
  int64_t sc_stride_batch, sc_stride_page, sc_stride_head;
  // INT4 cache: codes behind k / v (strides in bytes), eight fp16 parameters per row and tensor; q and the output are fp16
  // or bf16 (bf16 above)
  int32_t int4;
  const __half* k_param;
  const __half* v_param;
  int64_t pa_stride_batch, pa_stride_page, pa_stride_token, pa_stride_head;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N));
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void lds128(uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d, uint32_t addr) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(addr));
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  if (BF16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
// one output element in the storage type
template <bool BF16>
__device__ __forceinline__ void store_half(__half* dst, float x) {
  if (BF16) *reinterpret_cast<__nv_bfloat16*>(dst) = __float2bfloat16_rn(x);
  else *dst = __float2half_rn(x);
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
  return r;
}

// Merges the (maximum, sum, O) of a CTA's warps, which lie in shared memory, and writes the result, or the split's partial.
template <bool HAS_V, bool BF16>
__device__ __forceinline__ void merge_warps(const DecodeParams& p, const float* sm_m, const float* sm_l, const float* sm_o,
                                            int WARPS, int b, int g, int split) {
  for (int t = threadIdx.x; t < kHg * kD; t += WARPS * 32) {
    const int h = t / kD, d = t % kD;
    float M = -INFINITY;
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, sm_m[w * kHg + h]);
    float L = 0.f, O = 0.f;
    for (int w = 0; w < WARPS; ++w) {
      float mw = sm_m[w * kHg + h];
      float f = (mw == -INFINITY) ? 0.f : exp2f(mw - M);
      L += sm_l[w * kHg + h] * f;
      if (HAS_V) O += sm_o[(w * kHg + h) * kD + d] * f;
    }
    const int64_t bh = (int64_t)b * p.H + g * kHg + h;
    if (p.num_splits == 1) {
      if (HAS_V) store_half<BF16>(p.out + bh * kD + d, L > 0.f ? O / L : 0.f);
      if (d == 0 && p.lse2) p.lse2[bh] = L > 0.f ? M + log2f(L) : -INFINITY;
    } else {
      const int64_t slot = bh * p.num_splits + split;
      if (HAS_V) p.ws_o[slot * kD + d] = O;
      if (d == 0) { p.ws_m[slot] = M; p.ws_l[slot] = L; }
    }
  }
}

// Decode attention over a 4-bit cache (decode4.cu); dense: all keys of a sequence, with the logits written
cudaError_t launch_attn4(const DecodeParams& p, bool dense, bool has_v, dim3 grid, cudaStream_t st);
int init_decode4();

}  // namespace kb200
