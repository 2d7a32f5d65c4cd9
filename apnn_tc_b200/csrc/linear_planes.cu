// Matrix product of 16-bit float activations and weights held as bit planes, with bias, activation and residual in its
// epilogue.
#include <cmath>

#include "kv4.cuh"
#include "tc5_common.cuh"

namespace apnn {
namespace {

using namespace tc5;

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
};

__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case APNN_ACT_RELU: return v > 0.0f ? v : (v == v ? 0.0f : v);
    case APNN_ACT_SILU: return v / (1.0f + expf(-v));
    case APNN_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678f));
    case APNN_ACT_GELU_TANH: return 0.5f * v * (1.0f + tanhf(0.79788456f * (v + 0.044715f * v * v * v)));
    default: return v;
  }
}

// One warp per output element.
template <bool BF16>
__global__ void __launch_bounds__(256) linear_rows_kernel(const LinearParams p) {
  const int lane = threadIdx.x & 31;
  const long long n = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int m = blockIdx.y;
  grid_dependency_wait();
  if (p.status_flag && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *p.status_flag = 0;
  if (n >= p.N) return;
  float sum = 0.0f;
  for (int w = 0; w < p.kwords; w++) {
    const int k = w * 32 + lane;
    uint32_t level = 0;
    for (int b = 0; b < p.wbits; b++) level |= ((__ldg(p.W + b * p.plane_words + n * p.kwords + w) >> (31 - lane)) & 1u) << b;
    if (k < p.K) sum += unpack2<BF16>(p.X[m * p.ldx + k]).x * ((float)level - p.zero);
  }
#pragma unroll
  for (int d = 1; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane != 0) return;
  float v = activate(fmaf(sum, __ldg(p.scale + n), p.bias ? __ldg(p.bias + n) : 0.0f), p.act);
  if (p.residual) v += p.out_f32 ? static_cast<const float*>(p.residual)[m * p.ldr + n] : unpack2<BF16>(static_cast<const uint16_t*>(p.residual)[m * p.ldr + n]).x;
  if (p.out_f32) static_cast<float*>(p.out)[m * p.ldo + n] = v;
  else static_cast<uint16_t*>(p.out)[m * p.ldo + n] = (uint16_t)pack2<BF16>(v, 0.0f);
}

}  // namespace
}  // namespace apnn

using namespace apnn;

extern "C" apnn_status apnn_linear_planes(void* stream, int wbits, const void* W, const void* X, void* Out, int M, int N, int K,
                                          const apnn_linear_desc* d, int* status_flag) {
  if (!W || !X || !Out || !d || d->struct_size != sizeof(apnn_linear_desc) || !d->scale) return APNN_ERR_INVALID_ARG;
  if (M <= 0 || N <= 0 || K <= 0) return APNN_ERR_INVALID_ARG;
  if (d->x_type != APNN_TYPE_BF16 && d->x_type != APNN_TYPE_FP16) return APNN_ERR_INVALID_ARG;
  if (d->out_type != d->x_type && d->out_type != APNN_TYPE_FP32) return APNN_ERR_INVALID_ARG;
  if (d->activation < APNN_ACT_NONE || d->activation > APNN_ACT_GELU_TANH) return APNN_ERR_INVALID_ARG;
  if (!(d->zero >= 0.0f && d->zero <= 15.0f) || d->zero * 2.0f != std::floor(d->zero * 2.0f)) return APNN_ERR_INVALID_ARG;
  if (d->ldx < K || d->ldo < N || (d->residual && d->ldr < N)) return APNN_ERR_INVALID_ARG;
  if (wbits < 1 || wbits > 4) return APNN_ERR_UNSUPPORTED;
  const uintptr_t element = d->out_type == APNN_TYPE_FP32 ? 3u : 1u;
  if (((reinterpret_cast<uintptr_t>(W) | reinterpret_cast<uintptr_t>(X)) & 15u) != 0 || d->ldx % 8 != 0 ||
      ((reinterpret_cast<uintptr_t>(Out) | reinterpret_cast<uintptr_t>(d->residual)) & element) != 0 ||
      ((reinterpret_cast<uintptr_t>(d->scale) | reinterpret_cast<uintptr_t>(d->bias) | reinterpret_cast<uintptr_t>(status_flag)) & 3u) != 0)
    return APNN_ERR_ALIGNMENT;
  LinearParams p = {};
  p.W = static_cast<const uint32_t*>(W);
  p.X = static_cast<const uint16_t*>(X);
  p.out = Out;
  p.scale = d->scale;
  p.bias = d->bias;
  p.residual = d->residual;
  p.ldx = d->ldx;
  p.ldo = d->ldo;
  p.ldr = d->ldr;
  p.M = M;
  p.N = N;
  p.K = K;
  p.kwords = (K + 127) / 128 * 4;
  p.plane_words = (long long)N * p.kwords;
  p.wbits = wbits;
  p.act = d->activation;
  p.out_f32 = d->out_type == APNN_TYPE_FP32;
  p.zero = d->zero;
  p.status_flag = status_flag;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((N + 7) / 8), (unsigned)M, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  cfg.numAttrs = pdl_attribute(attr);
  cfg.attrs = attr;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, d->x_type == APNN_TYPE_BF16 ? linear_rows_kernel<true> : linear_rows_kernel<false>, p);
  return e == cudaSuccess ? APNN_OK : cuda_fail(e, "linear_rows_kernel");
}
