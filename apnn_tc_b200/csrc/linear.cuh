// The product over weight planes: parameters, activations and the store that its kernels share.
#pragma once
#include "kv4.cuh"
#include "spread.cuh"
#include "tc5_common.cuh"

namespace apnn {

struct LinearParams {
  const uint32_t* W;
  const uint16_t* X;
  void* out;
  const float* scale;
  const float* bias;
  const void* residual;
  long long ldx, ldo, ldr, plane_words;
  int M, N, K, kwords, wbits, act, out_f32;
  float zero;
  int* status_flag;
  int split;       // few rows: blocks of a cluster, which share K
};

// 1 / (1 + exp(-x)) to a few units of 2^-23: one exponential and one reciprocal instruction
__device__ __forceinline__ float logistic(float x) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}
__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case APNN_ACT_RELU: return v > 0.0f ? v : (v == v ? 0.0f : v);
    case APNN_ACT_SILU: return v * logistic(v);
    case APNN_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678f));
    case APNN_ACT_GELU_TANH: return v * logistic(1.5957691f * (v + 0.044715f * v * v * v));      // (1 + tanh u) / 2 = logistic(2 u)
    default: return v;
  }
}

// The epilogue of one output element.
template <bool BF16>
__device__ __forceinline__ void store_element(const LinearParams& p, long long m, long long n, float sum, float scale, float bias) {
  float v = activate(fmaf(sum, scale, bias), p.act);
  if (p.out_f32) {
    if (p.residual) v += static_cast<const float*>(p.residual)[m * p.ldr + n];
    static_cast<float*>(p.out)[m * p.ldo + n] = v;
  } else {
    if (p.residual) v += unpack2<BF16>(static_cast<const uint16_t*>(p.residual)[m * p.ldr + n]).x;
    static_cast<uint16_t*>(p.out)[m * p.ldo + n] = (uint16_t)pack2<BF16>(v, 0.0f);
  }
}

// More than a few rows (linear_tile.cu): blocks that share a tile (1 or 2), rows of X in it, blocks of a cluster that share its K.
struct LinearPlan {
  int ctas, tn, split;
};
LinearPlan linear_tile_plan(int M, int N, int kwords);
apnn_status linear_tile(cudaStream_t s, const LinearParams& p, bool bf16);

}  // namespace apnn
