// Shared by the kernels of the gated feed-forward block (ffn.cu, ffn_tc.cu, ffn_few.cu, ffn_token.cu).
#pragma once

#include "pack8.cuh"

namespace dsalt {
namespace ffn {

constexpr float LOG2E = 1.4426950408889634f;
// of numbers of at least 1, to 2^-23; of infinity 0
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// act(g) and act'(g) in fp32. silu: g p with p = 1 / (1 + e^-g); gelu: g p with p the normal
// distribution's share below g. By CUDA's functions, or FAST (the tensor cores' epilogues, whose results are rounded
// to 16 bits). FAST gelu: with the exponential that the derivative needs as well, the share below -x as e^(-x^2/2) t P(t), t = 1 / (1 + 0.302 x), the
// form of Hastings' approximations. P has six terms, fitted by linear programming for its relative error, which stays
// below 2^-16 where the share is small and below 2^-18 for x < 2 (Hastings' own five terms, Abramowitz
// and Stegun 7.1.26, hold 7.5e-8 of the whole, which at g = -5 is 1.6e-3 of the value: three half steps of fp16).
// CUDA's function takes about three times the instructions (first epilogue of 1999 x 768 -> 2048: 30 us against 20).
__device__ __forceinline__ float share_below(float g, float e) {  // e = exp(-g^2 / 2)
  const float t = reciprocal(fmaf(0.302f, fabsf(g), 1.f));
  float p = fmaf(-0.07876049727f, t, 0.2148901522f);
  p = fmaf(p, t, -0.01635385491f);
  p = fmaf(p, t, 0.1448939443f);
  p = fmaf(p, t, 0.1144450083f);
  p = fmaf(p, t, 0.1208847687f);
  const float tail = e * t * p;
  return g < 0.f ? tail : 1.f - tail;
}
// p = 1 / (1 + e^-g) and 1 - p. FAST: p to some 2^-21 of itself near 0; the argument's rounding grows with it, to 2^-20
// at -20 and 2^-18 at -80; below the normal range 0.
template <bool FAST>
__device__ __forceinline__ float2 sigmoid(float g) {
  if constexpr (FAST) {
    const float p = reciprocal(1.f + ex2_approx(-LOG2E * g));
    return make_float2(p, 1.f - p);
  } else {
    const float e = expf(-fabsf(g)), large = 1.f / (1.f + e), small = e * large;
    return g < 0.f ? make_float2(small, large) : make_float2(large, small);
  }
}
template <int ACT, bool FAST>
__device__ __forceinline__ float activate(float g) {
  if constexpr (ACT == DSALT_ACT_SILU) return g * sigmoid<FAST>(g).x;
  else if constexpr (FAST) return g * share_below(g, ex2_approx(-0.5f * LOG2E * g * g));
  else return g * normcdff(g);
}
template <int ACT, bool FAST>
__device__ __forceinline__ void activate_grad(float g, float& a, float& da) {
  if constexpr (ACT == DSALT_ACT_SILU) {
    const float2 p = sigmoid<FAST>(g);
    a = g * p.x;
    da = fmaf(a, p.y, p.x);
  } else {
    float e, p;
    if constexpr (FAST) {
      e = ex2_approx(-0.5f * LOG2E * g * g);
      p = share_below(g, e);
    } else {
      const float square = g * g;  // what its rounding leaves out counts where it is large
      e = expf(-0.5f * square);
      if (e > 0.f) e = fmaf(-0.5f * fmaf(g, g, -square), e, e);
      p = normcdff(g);
    }
    a = g * p;
    da = fmaf(g * 0.3989422804014327f, e, p);
  }
}

// What a backward pass of 16-bit inputs reads of gate's and up's sums: 24 of their 32 bits, each value by itself (codes
// with a scale for 32 neighbours, of 16 bits, held a feature 2^10 times smaller than one beside it worse than
// its own type does, and none beside an infinity). Three planes of 16 bits: gate's upper halves, up's, and both third bytes.
// The fourth byte is cut off: sums of at most 16 significant bits are held exactly, others are off by less than
// 2^-15 of themselves, towards zero (the mean, 2^-16, is far below the rounding of their gradients to 16 bits).
__device__ __forceinline__ uint32_t upper_halves(float a, float b) {
  return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
}
__device__ __forceinline__ uint32_t third_bytes(float gate, float up) {  // in the lower half
  return __byte_perm(__float_as_uint(gate), __float_as_uint(up), 0x0051);
}
// gate's (UP = 0) or up's two values of a pair of columns
template <int UP>
__device__ __forceinline__ float2 held24(uint32_t upper, uint32_t third) {
  const uint32_t t = UP ? __byte_perm(third, 0u, 0x4341) : third & 0x00ff00ffu;  // byte, zero, byte, zero
  return make_float2(__uint_as_float(__byte_perm(upper, t, 0x1045)), __uint_as_float(__byte_perm(upper, t, 0x3267)));
}

inline int64_t pitch_of(int64_t d_ff) { return (d_ff + GROUP8 - 1) / GROUP8 * GROUP8; }

// One call's sizes and operands. Rows of h, dg, du and of what is kept are `pitch` values long.
struct Ffn {
  int dtype, act, keep;
  int64_t T;
  int d, F, d_out;
  int64_t pitch;
  const void* w_gate;
  const void* w_up;
  const void* w_down;
  const void* x;
  int64_t x_stride;
  void* kept;       // [3, T, pitch]: gate, up and h in fp32, or gate and up in 24 bits; [2, T, pitch] codes of 8
  uint8_t* exps;    // [2, pitch / 32, T] of codes
  // forward
  void* y;
  void* h;          // [T, pitch]
  // backward
  const void* dy;
  int64_t dy_stride;
  void* dg;
  void* du;
  void* dx;
  void* dw_gate;
  void* dw_up;
  void* dw_down;
  float* wide;      // [T, pitch] fp32 once or twice (the path of ffn.cu's own products)
  cudaStream_t stream;
};

// 16-bit types whose sizes are multiples of 8 and whose operands' rows are 16-byte aligned
int run_tensor_cores(const Ffn& f, bool backward);
int forward_tokens(const Ffn& f);  // up to 16 tokens, nothing kept
int forward_few(const Ffn& f);     // few tokens, nothing kept

}  // namespace ffn
}  // namespace dsalt
