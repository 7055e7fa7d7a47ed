// KV-cache write path: optional per-head RMS norm of Q and K (Qwen3), rotary position embedding of Q
// and K (the half-rotation convention of the Hugging Face Llama / Qwen3 models), and the append of the
// new K / V rows into the paged (or contiguous) cache — one pass over the new tokens, so that the
// attention kernels find the cache in the layout they read, without the transposes and
// `.contiguous()` copies the reference's strategy pays before every kernel call
// (strategies/EfficientKascadeStrategy.py:144-150).  Bound by HBM: each new row is read once and
// written once.
//
// Arithmetic follows the Hugging Face modules step by step, in the model's type (fp16 or bf16), so that
// results agree to the last bit wherever sin / cos round the same way: the norm is computed in fp32 and
// rounded to that type before the gain is applied (LlamaRMSNorm / Qwen3RMSNorm), cos and sin are computed
// in fp32 from position * inv_freq[i] (the model's own inverse-frequency table, so every rope-scaling
// variant is covered), scaled and rounded to that type, and  x * cos + rotate_half(x) * sin  is evaluated
// in that type with a rounding after each product and after the sum (apply_rotary_pos_emb).
//
// Tokens with positions of their own (kb200_kv_write_at) are not the modules' arithmetic repeated: a cache that rows have
// left, or images and video with several axes, continue at positions far beyond the cache, where an angle formed in fp32 is
// off by up to pos 2^-24 and each rounding to bf16 costs as much again.  There the angle is formed and reduced in 64 bits
// (a few instructions of 64 of the threads of a CTA), norm and rotation are computed in fp32 and rounded once.
#include <cuda_bf16.h>

#include <climits>
#include <type_traits>

#include "common.cuh"

namespace kb200 {

struct KvWriteParams {
  const __half* q_in; __half* q_out; int64_t q_sb, q_st, q_sh;      // [B, T, H, D] views (q_out contiguous)
  const __half* k_new; int64_t k_sb, k_st, k_sh;                     // [B, T, G, D]
  const __half* v_new; int64_t v_sb, v_st, v_sh;
  const int32_t* start_pos;                                           // [B] cache length before the append
  const int32_t* n_new;                                               // [B] or null (= T)
  __half* k_cache; __half* v_cache;
  int64_t c_sb, c_sp, c_st, c_sh;                                     // cache strides (batch, page, token, head)
  const int32_t* block_table; int bt_stride; int page_shift, page_mask;
  const __half* q_gain; const __half* k_gain; float eps;              // RMS-norm gains [D] or null
  // FP8 (e4m3) cache: a row is stored as value / scale of its (page, KV head); strides of the cache in bytes
  const float* k_scale; const float* v_scale; int64_t s_sb, s_sp, s_sh;
  const float* inv_freq; float rope_scale;                            // [D/2] inverse frequencies or null (no rotary)
  int B, T, H, G;
  // INT4 cache: codes behind k_cache / v_cache (strides of the cache in bytes), eight fp16 parameters per row
  __half* k_param; __half* v_param; int64_t pa_sb, pa_sp, pa_st, pa_sh;
  // positions of their own: [axes, B, T], the axis of every rotary pair [D/2] or null (the first), and where the position on
  // the first axis is noted per cache row, [B, rows], or null
  const int32_t* positions; int64_t ps_axis, ps_b; const int32_t* pair_axis; int axes;
  int32_t* token_positions; int64_t tp_sb; int tp_rows;
  int tokens, chunks;                                                 // kv_append_kernel: tokens of a CTA, CTAs of a sequence
};

// One CTA per (sequence, new token): the token's 64 (cos, sin) pairs are computed once and shared by all
// its heads; a row of 128 values is handled by 8 lanes (lane c holds elements 8c..8c+7 and
// 64+8c..64+8c+7: the two elements a rotation pairs up sit in the same lane, 16-byte loads and stores),
// a warp takes four rows at a time.
constexpr int kKvWriteThreads = 192;

// The storage type of the activations and the cache: fp16, or bf16 (the pointers of KvWriteParams are then
// bf16 in disguise).  Every rounding step is the one the Hugging Face modules take in that type.
template <bool BF16> struct Pair { using T = __half2; using S = __half; };
template <> struct Pair<true> { using T = __nv_bfloat162; using S = __nv_bfloat16; };
__device__ __forceinline__ float2 to_f2(__half2 x) { return __half22float2(x); }
__device__ __forceinline__ float2 to_f2(__nv_bfloat162 x) { return __bfloat1622float2(x); }
template <bool BF16> __device__ __forceinline__ typename Pair<BF16>::T from_f2(float a, float b) {
  if constexpr (BF16) return __floats2bfloat162_rn(a, b);
  else return __floats2half2_rn(a, b);
}
template <bool BF16> __device__ __forceinline__ typename Pair<BF16>::S from_f(float a) {
  if constexpr (BF16) return __float2bfloat16_rn(a);
  else return __float2half_rn(a);
}

// eight values of the storage type (four pairs) -> eight e4m3 bytes of value / scale (fp32 division, saturating,
// round to nearest even)
template <typename H2>
__device__ __forceinline__ uint2 quantize8(const H2* x, float scale) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 a = to_f2(x[2 * i]), b = to_f2(x[2 * i + 1]);
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(lo) : "f"(a.y / scale), "f"(a.x / scale));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(hi) : "f"(b.y / scale), "f"(b.x / scale));
    w[i] = (uint32_t)lo | ((uint32_t)hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

// the norm's second half and the rotation as the Hugging Face modules round them; eight lanes per row, r = 1 / rms of the row
template <bool BF16>
__device__ __forceinline__ void module_norm(typename Pair<BF16>::T* lo, typename Pair<BF16>::T* hi, const __half* gain, float r, int c) {
  using H2 = typename Pair<BF16>::T;
  // x.float() * rsqrt(mean(x^2) + eps), rounded to the storage type, times the gain (a product in that type)
  const uint4 g_lo4 = reinterpret_cast<const uint4*>(gain)[c];
  const uint4 g_hi4 = reinterpret_cast<const uint4*>(gain + kD / 2)[c];
  const H2* g_lo = reinterpret_cast<const H2*>(&g_lo4);
  const H2* g_hi = reinterpret_cast<const H2*>(&g_hi4);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 a = to_f2(lo[e]), d2 = to_f2(hi[e]);
    lo[e] = __hmul2_rn(g_lo[e], from_f2<BF16>(a.x * r, a.y * r));
    hi[e] = __hmul2_rn(g_hi[e], from_f2<BF16>(d2.x * r, d2.y * r));
  }
}
template <bool BF16>
__device__ __forceinline__ void module_rotate(typename Pair<BF16>::T* lo, typename Pair<BF16>::T* hi, const typename Pair<BF16>::S* cos_s,
                                              const typename Pair<BF16>::S* sin_s, int c) {
  using H2 = typename Pair<BF16>::T;
  const uint4 cs4 = reinterpret_cast<const uint4*>(cos_s)[c];
  const uint4 sn4 = reinterpret_cast<const uint4*>(sin_s)[c];
  const H2* cs = reinterpret_cast<const H2*>(&cs4);
  const H2* sn = reinterpret_cast<const H2*>(&sn4);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    // first half:  x_lo * cos + (-x_hi) * sin ; second half:  x_hi * cos + x_lo * sin
    // (the _rn forms are never contracted into a fused multiply-add, which would skip a rounding)
    const H2 new_lo = __hadd2_rn(__hmul2_rn(lo[e], cs[e]), __hmul2_rn(__hneg2(hi[e]), sn[e]));
    const H2 new_hi = __hadd2_rn(__hmul2_rn(hi[e], cs[e]), __hmul2_rn(lo[e], sn[e]));
    lo[e] = new_lo;
    hi[e] = new_hi;
  }
}

// CTAS: CTAs per SM that the registers have to allow (0: left to the compiler); see launch_kv_write
template <bool BF16, bool FP8, int CTAS>
__global__ void __launch_bounds__(kKvWriteThreads, CTAS) kv_write_kernel(const KvWriteParams p) {
  using H2 = typename Pair<BF16>::T;
  using H1 = typename Pair<BF16>::S;
  __shared__ __align__(16) H1 cos_s[kD / 2];
  __shared__ __align__(16) H1 sin_s[kD / 2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / p.T, t = blockIdx.x - b * p.T;
  const int n = p.n_new ? p.n_new[b] : p.T;
  if (t >= n) return;
  const int heads = p.H + 2 * p.G;                                   // Q heads, K heads, V heads
  const int c = lane & 7;
  // The rows a warp takes next are loaded before the current ones are worked on, the first ones before sin and cos: a
  // CTA lives for two or three such steps only, so a load that waits for the step before it is time without traffic.
  auto load_rows = [&](int h0, uint4& lo, uint4& hi) {
    const int h = min(h0 + (lane >> 3), heads - 1);
    const __half* src = h < p.H ? p.q_in + b * p.q_sb + t * p.q_st + h * p.q_sh
                      : h < p.H + p.G ? p.k_new + b * p.k_sb + t * p.k_st + (h - p.H) * p.k_sh
                                      : p.v_new + b * p.v_sb + t * p.v_st + (h - p.H - p.G) * p.v_sh;
    lo = reinterpret_cast<const uint4*>(src)[c];                     // elements 8c .. 8c+7
    hi = reinterpret_cast<const uint4*>(src + kD / 2)[c];            // elements 64+8c .. 64+8c+7
  };
  constexpr int kStep = (kKvWriteThreads / 32) * 4;
  uint4 next_lo = make_uint4(0u, 0u, 0u, 0u), next_hi = next_lo;
  if (warp * 4 < heads) load_rows(warp * 4, next_lo, next_hi);
  const int pos = p.start_pos[b] + t;
  if (p.inv_freq && tid < kD / 2) {
    float sn, cs;
    sincosf((float)pos * p.inv_freq[tid], &sn, &cs);
    cos_s[tid] = from_f<BF16>(cs * p.rope_scale);
    sin_s[tid] = from_f<BF16>(sn * p.rope_scale);
  }
  __syncthreads();
  for (int h0 = warp * 4; h0 < heads; h0 += kStep) {                 // uniform per warp
    const int h = min(h0 + (lane >> 3), heads - 1);
    const bool active = h0 + (lane >> 3) < heads;                    // the last group of rows may be partial
    const int kind = h < p.H ? 0 : (h < p.H + p.G ? 1 : 2);          // 0 = Q, 1 = K, 2 = V
    const int hh = kind == 0 ? h : (kind == 1 ? h - p.H : h - p.H - p.G);
    uint4 lo4 = next_lo, hi4 = next_hi;
    if (h0 + kStep < heads) load_rows(h0 + kStep, next_lo, next_hi);
    H2* lo = reinterpret_cast<H2*>(&lo4);
    H2* hi = reinterpret_cast<H2*>(&hi4);
    const __half* gain = kind == 0 ? p.q_gain : (kind == 1 ? p.k_gain : nullptr);
    // sum of squares of the row: all lanes of the warp take part in the shuffles, whatever their row is
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 a = to_f2(lo[e]), d2 = to_f2(hi[e]);
      ss += a.x * a.x + a.y * a.y + d2.x * d2.x + d2.y * d2.y;
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
    if (gain) {
      module_norm<BF16>(lo, hi, gain, rsqrtf(ss / kD + p.eps), c);
    }
    if (kind != 2 && p.inv_freq) {
      module_rotate<BF16>(lo, hi, cos_s, sin_s, c);
    }
    __half* dst;
    if (kind == 0) {
      dst = p.q_out + (((int64_t)b * p.T + t) * p.H + hh) * kD;
    } else {
      const int page = pos >> p.page_shift, slot = pos & p.page_mask;
      const int64_t phys = p.block_table ? (int64_t)p.block_table[(int64_t)b * p.bt_stride + page] : page;
      if (FP8) {
        if (active) {
          const float sc = (kind == 1 ? p.k_scale : p.v_scale)[b * p.s_sb + phys * p.s_sp + hh * p.s_sh];
          uint8_t* d8 = reinterpret_cast<uint8_t*>(kind == 1 ? p.k_cache : p.v_cache) + b * p.c_sb + phys * p.c_sp +
                        slot * p.c_st + hh * p.c_sh;
          reinterpret_cast<uint2*>(d8)[c] = quantize8(lo, sc);              // bytes 8c .. 8c+7
          reinterpret_cast<uint2*>(d8 + kD / 2)[c] = quantize8(hi, sc);     // bytes 64+8c .. 64+8c+7
        }
        continue;
      }
      dst = (kind == 1 ? p.k_cache : p.v_cache) + b * p.c_sb + phys * p.c_sp + slot * p.c_st + hh * p.c_sh;
    }
    if (active) {
      reinterpret_cast<uint4*>(dst)[c] = lo4;
      reinterpret_cast<uint4*>(dst + kD / 2)[c] = hi4;
    }
  }
}

// The rows loaded one step ahead take nine registers a thread, which is one resident CTA per SM less.  Where a warp has one
// step only (24 heads or fewer: appends without Q) nothing is there to load ahead, and with more CTAs than the SMs
// hold the missing CTA costs time: those are compiled for seven per SM.  Measured before the loads ahead / with them /
// as it is now, us without Q, with and without rotary table: 32768 tokens 61.0 / 66.5 / 58.3, 56.0 / 63.2 / 54.3; 16 x 600
// 20.7 / 22.0 / 19.2, 19.2 / 21.2 / 18.2; 64 tokens 2.45 / 2.51 / 2.51, 2.26 / 2.26 / 2.26.
template <bool BF16, bool FP8>
static void launch_kv_write(const KvWriteParams& p, int64_t blocks, cudaStream_t st) {
  if (p.H + 2 * p.G <= kKvWriteThreads / 32 * 4 && blocks > 6ll * sm_count())
    kv_write_kernel<BF16, FP8, 7><<<(unsigned)blocks, kKvWriteThreads, 0, st>>>(p);
  else
    kv_write_kernel<BF16, FP8, 0><<<(unsigned)blocks, kKvWriteThreads, 0, st>>>(p);
}

// ---- appends that quantise to 4 bits, or whose tokens have positions of their own ---------------------
// pairs of fp32 numbers, for the two-element instructions: these kernels are bound by issue slots
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t sub2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("sub.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// What four lanes hold as four pieces each, exchanged: piece i of lane q becomes piece q of lane i.
template <typename T>
__device__ __forceinline__ void exchange4(T& a0, T& a1, T& a2, T& a3, int q) {
  auto swap = [](T& low, T& high, bool up, int with) {               // the lower lane's high piece for the upper lane's low one
    const T got = __shfl_xor_sync(0xFFFFFFFFu, up ? low : high, with);
    low = up ? got : low;
    high = up ? high : got;
  };
  swap(a0, a1, q & 1, 1);
  swap(a2, a3, q & 1, 1);
  swap(a0, a2, q & 2, 2);
  swap(a1, a3, q & 2, 2);
}

// the ends of a group of 32, as the row's own type or in fp32; a value that is not finite makes the upper end infinite or a NaN
template <bool BF16>
__device__ __forceinline__ void group_ends(const uint4* v, float& mn, float& mx) {
  using H2 = typename Pair<BF16>::T;
  const H2* h = reinterpret_cast<const H2*>(v);
  H2 least = h[0], most = h[0];
#pragma unroll
  for (int e = 1; e < 16; ++e) {
    least = __hmin2(least, h[e]);
    most = __hmax2_nan(most, h[e]);
  }
  const float2 lo = to_f2(least), hi = to_f2(most);
  mn = fminf(lo.x, lo.y);
  mx = hi.x == hi.x && hi.y == hi.y && mn > -INFINITY ? fmaxf(hi.x, hi.y) : INFINITY;
}
__device__ __forceinline__ void group_ends(const uint64_t* x, float& mn, float& mx) {
  uint64_t bad = 0;
  mn = INFINITY;
  mx = -INFINITY;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float2 v = unpack2(x[e]);
    mn = fminf(mn, fminf(v.x, v.y));
    mx = fmaxf(mx, fmaxf(v.x, v.y));
    bad = fma2(x[e], 0, bad);                                                  // a NaN if one is not finite
  }
  const float2 b = unpack2(bad);
  if (!(b.x + b.y == 0.f)) mx = INFINITY;
}

// The 4-bit form of a group of 32 values x whose ends are mn, mx:
//   z = fp16(min), s = fp16((max - z) / 15), c = round((x - z) / s) clamped to 0..15, half to even.
// Values saturate at +-65504, what fp16 can hold; a group with a value that is not finite gets z = NaN.  words: eight
// codes each, the lowest nibble first.
// A quotient is a product with 1 / s in two parts (good to 2^-44 together), rounded once: so quotients that are a number of 24 bits
// come out as that number, halves among them, and are rounded by adding 1.5 2^23.  (Halves are not rare, 0.07 % of bf16 values,
// because x, z and s have few bits; testing for them took as long as the division.)  The eight sums add up to the packed codes
// and a constant.  Clamping is needed only where fp16 rounds an end by a good part of a step.
__device__ __forceinline__ void quantize_int4(const uint64_t* x, float mn, float mx, uint32_t* words, __half& sh, __half& zh) {
  const bool fine = mx < INFINITY;
  zh = __float2half_rn(fine ? fminf(fmaxf(mn, -65504.f), 65504.f) : NAN);
  const float z = __half2float(zh);
  // (max - z) / 15, rounded once, in the same way (checked for every significand)
  const float span = fmaxf(fminf(mx, 65504.f) - z, 0.f), q0 = span * (1.f / 15.f);
  sh = __float2half_rn(fine ? fmaf(fmaf(-15.f, q0, span), 1.f / 15.f, q0) : 0.f);
  const float s = __half2float(sh);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(inv) : "f"(s));
  constexpr float kMagic = 12582912.f;                                          // 1.5 2^23: sums are rounded to whole numbers
  const float rest = fmaf(-s, inv, 1.f) * inv;                                  // (of s = 0 both are no numbers: clamped)
  const uint64_t minus_z2 = pack2(-z, -z), inv2 = pack2(inv, inv), rest2 = pack2(rest, rest), magic2 = pack2(kMagic, kMagic);
  const bool clamp = !(mn - z > -0.4f * s && mx - z < 15.4f * s);               // (also where s is 0, or z a NaN)
  float u[32];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint64_t a = add2(x[e], minus_z2);
    const float2 v = unpack2(add2(fma2(a, inv2, mul2(a, rest2)), magic2));
    u[2 * e] = v.x;
    u[2 * e + 1] = v.y;
  }
  if (__any_sync(0xFFFFFFFFu, clamp)) {                                         // (a branch: rarely taken, and long)
#pragma unroll
    for (int e = 0; e < 32; ++e)                                                // a NaN becomes 0, and so does all of it where s is 0
      if (clamp) u[e] = fminf(fmaxf(s > 0.f ? u[e] : 0.f, kMagic), kMagic + 15.f);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w = 0u - 0x4B400000u * 0x11111111u;                                // 0x4B400000: the bits of kMagic
#pragma unroll
    for (int e = 0; e < 8; ++e) w += __float_as_uint(u[8 * i + e]) << (4 * e);
    words[i] = w;
  }
}

// How a row is stored
constexpr int kSame = 0, kFp8 = 1, kInt4 = 2;
constexpr int kAppendThreads = 256;
constexpr int kAppendTokens = 4;                                               // tokens of a CTA at most

// Four lanes take an item: the K and the V row of a (token, KV head), whose places in the cache are the same, or two Q rows of a
// token.  To be normalised and rotated, lane q has the values 8q .. 8q+7 of each of a row's four groups of 32: the two that a rotation
// pairs up are in groups g and g + 2.  To be quantised, it has group q: what is done per group is then done once (with every group
// spread over the four lanes 32768 rows took 53 us).  Rows that nothing turns are loaded that way, the others are exchanged, and so are the
// codes, of which a lane stores one piece of 16 bytes per row.  A CTA takes p.tokens tokens; its first items are loaded before the
// angles are computed.  AT: positions of their own.  Quantising is bounded to 80 registers: with 64 / 118, 32768 rows take 52 / 46
// us, so 44.
template <bool BF16, int STORE, bool AT>
__global__ void __launch_bounds__(kAppendThreads, STORE == kInt4 ? 3 : 0) kv_append_kernel(const KvWriteParams p) {
  using H2 = typename Pair<BF16>::T;
  using Angle = typename std::conditional<AT, float, typename Pair<BF16>::S>::type;
  __shared__ __align__(16) Angle cos_s[kAppendTokens][kD / 2];
  __shared__ __align__(16) Angle sin_s[kAppendTokens][kD / 2];
  __shared__ int64_t page_s[kAppendTokens];
  __shared__ int slot_s[kAppendTokens];
  const int tid = threadIdx.x, q = tid & 3;
  const int per = p.G + (p.H + 1) / 2, items = p.tokens * per;       // items of a token: KV heads first, then pairs of Q heads
  const int b = blockIdx.x / p.chunks, t0 = (blockIdx.x - b * p.chunks) * p.tokens;
  const int t_end = p.n_new ? min(p.n_new[b], p.T) : p.T;
  const bool turns = p.k_gain || p.inv_freq;                          // K rows are normalised or rotated
  for (int item0 = 0; item0 < items; item0 += blockDim.x >> 2) {     // uniform for the CTA
    const int item = item0 + (tid >> 2);
    const int i = (item >= per) + (item >= 2 * per) + (item >= 3 * per), h = item - i * per;
    static_assert(kAppendTokens == 4, "three comparisons");
    const int t = t0 + i;
    const bool active = item < items && t < t_end;
    const bool kv = h < p.G;
    const int head = kv ? h : 2 * (h - p.G);
    const bool two = kv || head + 1 < p.H;
    uint4 row[2][4];                                                    // (all lanes take part in the shuffles)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const __half* src = !kv ? p.q_in + b * p.q_sb + t * p.q_st + (head + r) * p.q_sh
                              : r == 0 ? p.k_new + b * p.k_sb + t * p.k_st + head * p.k_sh
                                       : p.v_new + b * p.v_sb + t * p.v_st + head * p.v_sh;
      const bool whole = STORE == kInt4 && kv && !(r == 0 && turns);
#pragma unroll
      for (int g = 0; g < 4; ++g)
        row[r][g] = active && (r == 0 || two) ? reinterpret_cast<const uint4*>(src)[whole ? 4 * q + g : 4 * g + q]
                                              : make_uint4(0u, 0u, 0u, 0u);
    }
    if (item0 == 0) {
      // the tokens' places in the cache, and their angles
      for (int at = tid; at < p.tokens * (p.inv_freq ? kD / 2 : 1); at += blockDim.x) {
        const int j = p.inv_freq ? at / (kD / 2) : at, pair = p.inv_freq ? at % (kD / 2) : 0;
        if (t0 + j >= t_end) continue;
        const int pos = p.start_pos[b] + t0 + j;
        const int32_t* own = AT ? p.positions + b * p.ps_b + t0 + j : nullptr;
        if (pair == 0) {
          const int page = pos >> p.page_shift;
          page_s[j] = p.block_table ? (int64_t)p.block_table[(int64_t)b * p.bt_stride + page] : page;
          slot_s[j] = pos & p.page_mask;
          if (AT && p.token_positions && pos < p.tp_rows) p.token_positions[b * p.tp_sb + pos] = own[0];
        }
        if (!p.inv_freq) continue;
        float sn, cs;
        if constexpr (AT) {
          const int axis = p.pair_axis ? min(max(p.pair_axis[pair], 0), p.axes - 1) : 0;
          constexpr double kTurns = 0.1591549430918953357689;          // 1 / (2 pi)
          const double turns = (double)own[axis * p.ps_axis] * (double)p.inv_freq[pair] * kTurns;
          sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
          cos_s[j][pair] = cs * p.rope_scale;
          sin_s[j][pair] = sn * p.rope_scale;
        } else {
          sincosf((float)pos * p.inv_freq[pair], &sn, &cs);
          cos_s[j][pair] = from_f<BF16>(cs * p.rope_scale);
          sin_s[j][pair] = from_f<BF16>(sn * p.rope_scale);
        }
      }
      __syncthreads();
    }
    const int64_t phys = active ? page_s[i] : 0, slot = active ? slot_s[i] : 0;
    const int64_t place = b * p.c_sb + phys * p.c_sp + slot * p.c_st + head * p.c_sh;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const bool turn = p.inv_freq && (!kv || r == 0);
      const __half* gain = !kv ? p.q_gain : r == 0 ? p.k_gain : nullptr;
      const bool plain = AT && STORE != kInt4 && kv && r == 1;            // a V row that is stored as it is
      uint64_t x[16];                                                     // the row in fp32, four pairs per group
      auto widen = [&] {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const H2* v = reinterpret_cast<const H2*>(&row[r][g]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = to_f2(v[e]);
            x[4 * g + e] = pack2(f.x, f.y);
          }
        }
      };
      float inv_rms = 1.f;
      if (AT && !plain) widen();
      if (r == 0 ? p.q_gain || p.k_gain : p.q_gain != nullptr) {           // (uniform: the warp's rows are of either kind)
        uint64_t sq = 0;
        if constexpr (!AT) widen();
        if (!plain) {
#pragma unroll
          for (int e = 0; e < 16; ++e) sq = fma2(x[e], x[e], sq);
        }
        float ss = unpack2(sq).x + unpack2(sq).y;
        ss += __shfl_xor_sync(0xFFFFFFFFu, ss, 1);
        ss += __shfl_xor_sync(0xFFFFFFFFu, ss, 2);
        inv_rms = rsqrtf(ss / kD + p.eps);
      }
      if constexpr (AT) {
        if (!plain) {
          if (gain) {
            const uint64_t rms2 = pack2(inv_rms, inv_rms);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const uint4 g4 = reinterpret_cast<const uint4*>(gain)[4 * g + q];
              const H2* gv = reinterpret_cast<const H2*>(&g4);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = to_f2(gv[e]);
                x[4 * g + e] = mul2(x[4 * g + e], mul2(pack2(f.x, f.y), rms2));
              }
            }
          }
          if (turn) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                const ulonglong2 cs = *reinterpret_cast<const ulonglong2*>(&cos_s[i][32 * g + 8 * q + 2 * e]);
                const ulonglong2 sn = *reinterpret_cast<const ulonglong2*>(&sin_s[i][32 * g + 8 * q + 2 * e]);
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                  const uint64_t l = x[4 * g + e + f], h2 = x[8 + 4 * g + e + f], cv = f ? cs.y : cs.x, sv = f ? sn.y : sn.x;
                  x[4 * g + e + f] = sub2(mul2(l, cv), mul2(h2, sv));
                  x[8 + 4 * g + e + f] = fma2(l, sv, mul2(h2, cv));
                }
              }
            }
          }
          if (STORE != kInt4 || !kv) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              H2* v = reinterpret_cast<H2*>(&row[r][g]);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = unpack2(x[4 * g + e]);
                v[e] = from_f2<BF16>(f.x, f.y);
              }
            }
          }
        }
      } else {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          H2* lo = reinterpret_cast<H2*>(&row[r][g]);
          H2* hi = reinterpret_cast<H2*>(&row[r][g + 2]);
          if (gain) module_norm<BF16>(lo, hi, gain, inv_rms, 4 * g + q);
          if (turn) module_rotate<BF16>(lo, hi, cos_s[i], sin_s[i], 4 * g + q);
        }
      }
      uint32_t words[4], scale01 = 0u, scale23 = 0u, zero01 = 0u, zero23 = 0u;
      if constexpr (STORE == kInt4) {
        float mn, mx;
        if constexpr (AT) {
          if (r == 0 && turns) {
#pragma unroll
            for (int e = 0; e < 4; ++e) exchange4(x[e], x[4 + e], x[8 + e], x[12 + e], q);
          }
          group_ends(x, mn, mx);
        } else {
          if (r == 0 && turns) {                                          // (Q rows, which are stored as they are, keep theirs)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t w[4];
#pragma unroll
              for (int g = 0; g < 4; ++g) w[g] = reinterpret_cast<const uint32_t*>(&row[r][g])[e];
              exchange4(w[0], w[1], w[2], w[3], q);
#pragma unroll
              for (int g = 0; g < 4; ++g)
                if (kv) reinterpret_cast<uint32_t*>(&row[r][g])[e] = w[g];
            }
          }
          widen();
          group_ends<BF16>(row[r], mn, mx);
        }
        __half scale, zero;
        quantize_int4(x, mn, mx, words, scale, zero);
        exchange4(words[0], words[1], words[2], words[3], q);
        const uint32_t par = (uint32_t)__half_as_ushort(scale) | (uint32_t)__half_as_ushort(zero) << 16;
        const uint32_t next = __shfl_xor_sync(0xFFFFFFFFu, par, 1);
        scale01 = __byte_perm(par, next, 0x5410);                         // (as lanes 0 and 2 see them)
        zero01 = __byte_perm(par, next, 0x7632);
        scale23 = __shfl_xor_sync(0xFFFFFFFFu, scale01, 2);
        zero23 = __shfl_xor_sync(0xFFFFFFFFu, zero01, 2);
      }
      if (!active || (r && !two)) continue;
      __half* cache = r == 0 ? p.k_cache : p.v_cache;
      if (STORE == kSame || !kv) {
        uint4* dst = reinterpret_cast<uint4*>(kv ? cache + place : p.q_out + (((int64_t)b * p.T + t) * p.H + head + r) * kD);
#pragma unroll
        for (int g = 0; g < 4; ++g) dst[4 * g + q] = row[r][g];
      } else if constexpr (STORE == kInt4) {
        uint4 piece;                                                       // groups 0-3 of K; of V, whose pieces hold four values per
        if (r == 0) {                                                      // group, the low halves of the words, then the high ones
          piece = make_uint4(words[0], words[1], words[2], words[3]);
        } else {
          piece = make_uint4(__byte_perm(words[0], words[1], 0x5410), __byte_perm(words[2], words[3], 0x5410),
                             __byte_perm(words[0], words[1], 0x7632), __byte_perm(words[2], words[3], 0x7632));
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(cache) + place + q * 16) = piece;
        if (q == 0) {
          __half* dst = (r == 0 ? p.k_param : p.v_param) + b * p.pa_sb + phys * p.pa_sp + slot * p.pa_st + head * p.pa_sh;
          *reinterpret_cast<uint4*>(dst) = make_uint4(scale01, scale23, zero01, zero23);
        }
      } else {
        const float sc = (r == 0 ? p.k_scale : p.v_scale)[b * p.s_sb + phys * p.s_sp + head * p.s_sh];
        uint2* dst = reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(cache) + place);
#pragma unroll
        for (int g = 0; g < 4; ++g) dst[4 * g + q] = quantize8(reinterpret_cast<const H2*>(&row[r][g]), sc);
      }
    }
  }
}

// One warp per CTA where there are many tokens: then a CTA makes several passes, and while one waits for its rows or computes its angles
// the others on the SM work.  Few tokens: all items of a token at once.  us (and TB/s) for 32768 tokens of 8 KV heads to 4 bits 44
// (4.0; with rotary 53), of which quantising is 10 (storing sums of the values instead: 34).  16384 tokens of 32 + 8 heads with
// positions on three axes 71 (5.7; with norm 76).  With two / three warps per CTA those two take 76 / 83 and 85 / 91, and with all
// items at once 81 and 95; 64 tokens of 32 + 8 heads 5.7 with all items at once, 8.1 with two warps.
template <bool BF16, int STORE, bool AT>
static void launch_kv_append(KvWriteParams p, int64_t tokens, cudaStream_t st) {
  const int per = p.G + (p.H + 1) / 2;
  p.tokens = 1;
  while (p.tokens < kAppendTokens && p.tokens * 2 * per <= 16 && p.tokens * 2 <= p.T &&
         tokens >= (int64_t)p.tokens * 2 * 8 * sm_count())
    p.tokens *= 2;
  p.chunks = (p.T + p.tokens - 1) / p.tokens;
  const int threads = (p.tokens * per * 4 + 31) / 32 * 32, most = tokens > 8ll * sm_count() ? 32 : kAppendThreads;
  kv_append_kernel<BF16, STORE, AT><<<(unsigned)p.B * (unsigned)p.chunks, threads < most ? threads : most, 0, st>>>(p);
}
template <bool BF16>
static void launch_kv_append(const KvWriteParams& p, int store, int64_t tokens, cudaStream_t st) {
  if (store == kInt4 && p.positions) launch_kv_append<BF16, kInt4, true>(p, tokens, st);
  else if (store == kInt4) launch_kv_append<BF16, kInt4, false>(p, tokens, st);
  else if (store == kFp8) launch_kv_append<BF16, kFp8, true>(p, tokens, st);
  else launch_kv_append<BF16, kSame, true>(p, tokens, st);
}

// Rows of a 4-bit cache in 16 bits: four lanes per row.  Lane q loads 16 bytes of the codes of K, which are the values 8q .. 8q+7 of
// every group, and 16 of V, which are the same values in two pieces, and the eight parameters of either.
struct KvReadParams {
  const uint8_t* k; const uint8_t* v; int64_t c_sb, c_sp, c_st, c_sh;
  const __half* k_param; const __half* v_param; int64_t pa_sb, pa_sp, pa_st, pa_sh;
  const int32_t* block_table; int bt_stride; int page_shift, page_mask;
  const int32_t* seq_lens;
  __half* k_out; __half* v_out;                                       // [B, T, G, D]
  int G, rows, chunks;                                                // rows of a sequence (T G), CTAs that share them
};

// the eight values of a word of codes, the lowest nibble first: a code in the low bits of 2^23 is that number and the code.  Code 15
// of a group that reaches fp16's largest number can stand for more than that (s is rounded: 65536 for -65504 .. 65504): it
// saturates, as the row did on its way in; a NaN stays one.
template <bool BF16>
__device__ __forceinline__ uint4 from_codes(uint32_t w, uint64_t s2, uint64_t z2) {
  using H2 = typename Pair<BF16>::T;
  const uint64_t minus = pack2(-8388608.f, -8388608.f);
  H2 out[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint64_t c = pack2(__uint_as_float(((w >> (8 * e)) & 15u) | 0x4B000000u),
                             __uint_as_float(((w >> (8 * e + 4)) & 15u) | 0x4B000000u));
    const float2 v = unpack2(fma2(add2(c, minus), s2, z2));
    if constexpr (BF16) out[e] = from_f2<BF16>(v.x, v.y);
    else out[e] = __hmax2_nan(__hmin2_nan(from_f2<BF16>(v.x, v.y), __half2half2(__ushort_as_half(0x7BFF))), __half2half2(__ushort_as_half(0xFBFF)));
  }
  return *reinterpret_cast<uint4*>(out);
}

constexpr int kReadThreads = 256;
constexpr int kReadBlock = kReadThreads / 4;                              // rows of a CTA; a CTA stays within a sequence
// Bound by HBM: 32768 rows of 8 KV heads 31.4 us, 5.6 TB/s, the same with two or four rows per thread and with 64 or 128 threads.
template <bool BF16>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(const KvReadParams p) {
  const int b = blockIdx.x / p.chunks, row = (blockIdx.x - b * p.chunks) * kReadBlock + (threadIdx.x >> 2), q = threadIdx.x & 3;
  if (row >= p.rows) return;
  const int t = row / p.G, head = row - t * p.G;
  uint4 kw = make_uint4(0u, 0u, 0u, 0u), vw = kw, kp = kw, vp = kw;        // rows behind a sequence read as zeros
  if (t < p.seq_lens[b]) {
    const int lp = t >> p.page_shift, slot = t & p.page_mask;
    const int64_t page = p.block_table ? (int64_t)p.block_table[(int64_t)b * p.bt_stride + lp] : lp;
    const int64_t at = b * p.c_sb + page * p.c_sp + slot * p.c_st + head * p.c_sh + q * 16;
    const int64_t pa = b * p.pa_sb + page * p.pa_sp + slot * p.pa_st + head * p.pa_sh;
    kw = *reinterpret_cast<const uint4*>(p.k + at);
    vw = *reinterpret_cast<const uint4*>(p.v + at);
    kp = *reinterpret_cast<const uint4*>(p.k_param + pa);
    vp = *reinterpret_cast<const uint4*>(p.v_param + pa);
  }
  uint4* ko = reinterpret_cast<uint4*>(p.k_out + ((int64_t)b * p.rows + row) * kD) + q;      // group g: 16-byte piece 4 g + q
  uint4* vo = reinterpret_cast<uint4*>(p.v_out + ((int64_t)b * p.rows + row) * kD) + q;
  const uint32_t k_codes[4] = {kw.x, kw.y, kw.z, kw.w};
  const uint32_t v_codes[4] = {__byte_perm(vw.x, vw.z, 0x5410), __byte_perm(vw.x, vw.z, 0x7632), __byte_perm(vw.y, vw.w, 0x5410),
                               __byte_perm(vw.y, vw.w, 0x7632)};
  const __half* ks = reinterpret_cast<const __half*>(&kp);
  const __half* vs = reinterpret_cast<const __half*>(&vp);
  auto twice = [](__half x) { return pack2(__half2float(x), __half2float(x)); };
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    ko[4 * g] = from_codes<BF16>(k_codes[g], twice(ks[g]), twice(ks[4 + g]));
    vo[4 * g] = from_codes<BF16>(v_codes[g], twice(vs[g]), twice(vs[4 + g]));
  }
}

}  // namespace kb200

static int kv_write_call(const kb200_act_layout* q_in, void* q_out, const kb200_act_layout* k_new,
                         const kb200_act_layout* v_new, const int32_t* start_pos, const int32_t* n_new,
                         const kb200_kv_layout* kv, const void* q_norm_gain, const void* k_norm_gain,
                         float norm_eps, const float* inv_freq, float rope_scale, const kb200_positions* at, int batch,
                         int max_new, int num_q_heads, int num_kv_heads, void* stream) {
  using namespace kb200;
  KB_ENTRY(k_new ? k_new->ptr : nullptr, "kv_write: k_new");
  KB_REQUIRE(k_new && k_new->ptr && v_new && v_new->ptr && start_pos && kv && kv->k && kv->v,
             "kv_write: null pointer");
  KB_REQUIRE(batch >= 0 && max_new >= 0 && num_kv_heads > 0 && num_q_heads >= 0, "kv_write: bad sizes");
  const bool fp8 = kv->dtype == KB200_FP8_E4M3, int4 = kv->dtype == KB200_INT4;
  KB_REQUIRE((k_new->dtype == KB200_FP16 || k_new->dtype == KB200_BF16) && v_new->dtype == k_new->dtype &&
                 (fp8 || int4 || kv->dtype == k_new->dtype) && (!q_in || !q_in->ptr || q_in->dtype == k_new->dtype),
             "kv_write: q / k / v and the cache must all be fp16 or all bf16 (its arithmetic follows the Hugging Face "
             "modules step by step in that type; gains are in the same type), or the cache FP8 (e4m3) with scales, or INT4");
  if (int4) {
    if (check_int4(kv, true, "kv_write") != 0) return -1;
    KB_REQUIRE(kv->act_dtype == k_new->dtype, "kv_write: act_dtype of the INT4 cache (%d) is not the rows' type (%d)",
               kv->act_dtype, k_new->dtype);
  }
  if (at) {
    KB_REQUIRE(at->positions && at->axes >= 1, "kv_write_at: positions [axes, B, T] with at least one axis are required");
    KB_REQUIRE(!at->token_positions || at->token_rows >= 0, "kv_write_at: negative number of rows of token_positions");
  }
  KB_REQUIRE(!fp8 || (kv->k_scale && kv->v_scale), "kv_write: an FP8 cache needs k_scale / v_scale");
  const bool bf16 = k_new->dtype == KB200_BF16;
  KB_REQUIRE(kv->page_size >= 1 && (kv->page_size & (kv->page_size - 1)) == 0,
             "kv_write: page_size must be a power of two (got %d)", kv->page_size);
  KB_REQUIRE(!inv_freq || (reinterpret_cast<uintptr_t>(inv_freq) & 7) == 0, "kv_write: inv_freq must be 8-byte aligned");
  const bool with_q = q_in && q_in->ptr;
  KB_REQUIRE(!with_q || q_out, "kv_write: q_in given without q_out");
  auto aligned = [](const void* ptr, int64_t a, int64_t b2, int64_t c) {
    return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && a % 8 == 0 && b2 % 8 == 0 && c % 8 == 0;
  };
  KB_REQUIRE(aligned(k_new->ptr, k_new->stride_b, k_new->stride_t, k_new->stride_h) &&
                 aligned(v_new->ptr, v_new->stride_b, v_new->stride_t, v_new->stride_h) &&
                 (!with_q || aligned(q_in->ptr, q_in->stride_b, q_in->stride_t, q_in->stride_h)) &&
                 aligned(kv->k, kv->stride_batch, kv->stride_page, kv->stride_token) &&
                 aligned(kv->v, kv->stride_head, 0, 0),
             "kv_write: pointers must be 16-byte aligned and strides multiples of 8 elements");
  KB_REQUIRE(!fp8 || (kv->stride_batch % 16 == 0 && kv->stride_page % 16 == 0 && kv->stride_token % 16 == 0 &&
                      kv->stride_head % 16 == 0),
             "kv_write: strides of an FP8 cache must be multiples of 16 bytes");
  if (batch == 0 || max_new == 0) return 0;
  KvWriteParams p{};
  if (with_q) {
    p.q_in = static_cast<const __half*>(q_in->ptr);
    p.q_sb = q_in->stride_b; p.q_st = q_in->stride_t; p.q_sh = q_in->stride_h;
    p.q_out = static_cast<__half*>(q_out);
  }
  p.k_new = static_cast<const __half*>(k_new->ptr);
  p.k_sb = k_new->stride_b; p.k_st = k_new->stride_t; p.k_sh = k_new->stride_h;
  p.v_new = static_cast<const __half*>(v_new->ptr);
  p.v_sb = v_new->stride_b; p.v_st = v_new->stride_t; p.v_sh = v_new->stride_h;
  p.start_pos = start_pos;
  p.n_new = n_new;
  p.k_cache = static_cast<__half*>(const_cast<void*>(kv->k));
  p.v_cache = static_cast<__half*>(const_cast<void*>(kv->v));
  p.c_sb = kv->stride_batch; p.c_sp = kv->stride_page; p.c_st = kv->stride_token; p.c_sh = kv->stride_head;
  p.block_table = kv->block_table;
  p.bt_stride = kv->block_table_stride;
  int shift = 0;
  while ((1 << shift) < kv->page_size) ++shift;
  p.page_shift = shift;
  p.page_mask = kv->page_size - 1;
  p.k_scale = kv->k_scale;
  p.v_scale = kv->v_scale;
  p.s_sb = kv->scale_stride_batch; p.s_sp = kv->scale_stride_page; p.s_sh = kv->scale_stride_head;
  p.q_gain = static_cast<const __half*>(q_norm_gain);
  p.k_gain = static_cast<const __half*>(k_norm_gain);
  p.eps = norm_eps;
  p.inv_freq = inv_freq;
  p.rope_scale = rope_scale;
  if (int4) {
    p.k_param = static_cast<__half*>(const_cast<void*>(kv->k_param));
    p.v_param = static_cast<__half*>(const_cast<void*>(kv->v_param));
    p.pa_sb = kv->param_stride_batch; p.pa_sp = kv->param_stride_page; p.pa_st = kv->param_stride_token; p.pa_sh = kv->param_stride_head;
  }
  if (at) {
    p.positions = at->positions;
    p.ps_axis = at->stride_axis; p.ps_b = at->stride_batch;
    p.pair_axis = at->pair_axis;
    p.axes = at->axes;
    p.token_positions = at->token_positions;
    p.tp_sb = at->token_stride; p.tp_rows = at->token_rows;
  }
  p.B = batch; p.T = max_new; p.H = with_q ? num_q_heads : 0; p.G = num_kv_heads;
  const int64_t blocks = (int64_t)batch * max_new;                   // one CTA per (sequence, new token)
  KB_REQUIRE(blocks < (1ll << 31), "kv_write: too many tokens for one launch");
  cudaStream_t st = (cudaStream_t)stream;
  if (at || int4) {
    const int store = int4 ? kInt4 : fp8 ? kFp8 : kSame;
    if (bf16) launch_kv_append<true>(p, store, blocks, st);
    else launch_kv_append<false>(p, store, blocks, st);
    KB_CHECK_LAUNCH("kv_append_kernel");
    return 0;
  }
  if (bf16 && fp8) launch_kv_write<true, true>(p, blocks, st);
  else if (bf16) launch_kv_write<true, false>(p, blocks, st);
  else if (fp8) launch_kv_write<false, true>(p, blocks, st);
  else launch_kv_write<false, false>(p, blocks, st);
  KB_CHECK_LAUNCH("kv_write_kernel");
  return 0;
}

extern "C" int kb200_kv_write(const kb200_act_layout* q_in, void* q_out, const kb200_act_layout* k_new,
                              const kb200_act_layout* v_new, const int32_t* start_pos, const int32_t* n_new,
                              const kb200_kv_layout* kv, const void* q_norm_gain, const void* k_norm_gain,
                              float norm_eps, const float* inv_freq, float rope_scale, int batch, int max_new,
                              int num_q_heads, int num_kv_heads, void* stream) {
  return kv_write_call(q_in, q_out, k_new, v_new, start_pos, n_new, kv, q_norm_gain, k_norm_gain, norm_eps, inv_freq, rope_scale,
                       nullptr, batch, max_new, num_q_heads, num_kv_heads, stream);
}

extern "C" int kb200_kv_write_at(const kb200_act_layout* q_in, void* q_out, const kb200_act_layout* k_new,
                                 const kb200_act_layout* v_new, const int32_t* start_pos, const int32_t* n_new,
                                 const kb200_kv_layout* kv, const void* q_norm_gain, const void* k_norm_gain,
                                 float norm_eps, const float* inv_freq, float rope_scale, const kb200_positions* at, int batch,
                                 int max_new, int num_q_heads, int num_kv_heads, void* stream) {
  KB_REQUIRE(at, "kv_write_at: null pointer");
  return kv_write_call(q_in, q_out, k_new, v_new, start_pos, n_new, kv, q_norm_gain, k_norm_gain, norm_eps, inv_freq, rope_scale,
                       at, batch, max_new, num_q_heads, num_kv_heads, stream);
}

extern "C" int kb200_kv_read(const kb200_kv_layout* kv, const int32_t* seq_lens, void* k_out, void* v_out, int batch,
                             int max_len, int num_kv_heads, void* stream) {
  using namespace kb200;
  KB_ENTRY(k_out, "kv_read: k_out");
  KB_REQUIRE(kv && kv->k && kv->v && seq_lens && k_out && v_out, "kv_read: null pointer");
  KB_REQUIRE(kv->dtype == KB200_INT4, "kv_read: the cache is not INT4 (dtype code %d): its rows need no conversion", kv->dtype);
  if (check_int4(kv, true, "kv_read") != 0) return -1;
  KB_REQUIRE(batch >= 0 && max_len >= 0 && num_kv_heads > 0, "kv_read: bad sizes");
  KB_REQUIRE(kv->page_size >= 1 && (kv->page_size & (kv->page_size - 1)) == 0,
             "kv_read: page_size must be a power of two (got %d)", kv->page_size);
  KB_REQUIRE(((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) == 0,
             "kv_read: k_out and v_out must be 16-byte aligned");
  KvReadParams p{};
  if (batch == 0 || max_len == 0) return 0;
  const int64_t rows = (int64_t)max_len * num_kv_heads, chunks = (rows + kReadBlock - 1) / kReadBlock;
  KB_REQUIRE(rows <= INT_MAX - kReadBlock && batch * chunks < (1ll << 31), "kv_read: too many rows for one launch");
  p.rows = (int)rows;
  p.chunks = (int)chunks;
  p.k = static_cast<const uint8_t*>(kv->k);
  p.v = static_cast<const uint8_t*>(kv->v);
  p.c_sb = kv->stride_batch; p.c_sp = kv->stride_page; p.c_st = kv->stride_token; p.c_sh = kv->stride_head;
  p.k_param = static_cast<const __half*>(kv->k_param);
  p.v_param = static_cast<const __half*>(kv->v_param);
  p.pa_sb = kv->param_stride_batch; p.pa_sp = kv->param_stride_page; p.pa_st = kv->param_stride_token; p.pa_sh = kv->param_stride_head;
  p.block_table = kv->block_table;
  p.bt_stride = kv->block_table_stride;
  int shift = 0;
  while ((1 << shift) < kv->page_size) ++shift;
  p.page_shift = shift;
  p.page_mask = kv->page_size - 1;
  p.seq_lens = seq_lens;
  p.k_out = static_cast<__half*>(k_out);
  p.v_out = static_cast<__half*>(v_out);
  p.G = num_kv_heads;
  const unsigned blocks = (unsigned)(batch * chunks);
  if (kv->act_dtype == KB200_BF16) kv_read_kernel<true><<<blocks, kReadThreads, 0, (cudaStream_t)stream>>>(p);
  else kv_read_kernel<false><<<blocks, kReadThreads, 0, (cudaStream_t)stream>>>(p);
  KB_CHECK_LAUNCH("kv_read_kernel");
  return 0;
}
