// Attention over the 4-bit cache.
#include <cmath>

#include "kv4.cuh"
#include "tc5_common.cuh"

namespace apnn {
namespace {

using namespace tc5;

struct AttentionParams {
  Kv4View cache;
  Kv4Batch batch;
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  long long q_stride, out_stride;
  int q_heads, group, causal, window;
  float scale;
};

// One warp per row and query head, lanes over the head's elements.
template <bool BF16, int D>
__global__ void __launch_bounds__(128) kv4_attention_rows_kernel(const AttentionParams p) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = (int)(item / p.q_heads), h = (int)(item % p.q_heads);
  grid_dependency_wait();
  if (t >= p.batch.rows) return;
  const int b = sequence_of(p.batch.cu_q, p.batch.sequences, t, lane);
  if (b < 0) return;
  const int first = __ldg(p.batch.cu_q + b), len = __ldg(p.batch.kv_len + b);
  const int i = t - first;
  if (i >= p.batch.max_q) return;
  const int pos = len - (__ldg(p.batch.cu_q + b + 1) - first) + i;
  int end = len, begin = 0;
  if (p.causal) {
    end = min(end, pos + 1);
    if (p.window > 0) begin = max(0, pos + 1 - p.window);
  }
  end = (int)min((long long)end, (long long)p.batch.table_width << p.cache.page_shift);
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E; e++) {
    const uint32_t w = p.q[t * p.q_stride + (long long)h * D + lane * E + e];
    q[e] = unpack2<BF16>(w).x;
    o[e] = 0.0f;
  }
  float top = -INFINITY, sum = 0.0f;
  const long long codes = (long long)p.cache.page_size * (D / 2);
  for (int j = begin; j < end; j++) {
    const uint8_t* page = page_of(p.cache, p.batch, b, j);
    if (page == nullptr) continue;
    const uint8_t* head = page + (h / p.group) * p.cache.head_bytes;
    const int slot = j & (p.cache.page_size - 1);
    const float2 kp = unpack2<BF16>(*reinterpret_cast<const uint32_t*>(head + 2 * codes + slot * 4ll));
    const float2 vp = unpack2<BF16>(*reinterpret_cast<const uint32_t*>(head + 2 * codes + (p.cache.page_size + slot) * 4ll));
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int d = lane * E + e;
      const uint32_t n = (head[slot * (long long)(D / 2) + d / 2] >> (4 * (d & 1))) & 15u;
      s += q[e] * fmaf(kp.x, (float)n, kp.y);
    }
#pragma unroll
    for (int d = 1; d < 32; d *= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= p.scale;
    const float m = fmaxf(top, s);
    const float keep = top == -INFINITY ? 0.0f : expf(top - m), w = expf(s - m);
    sum = sum * keep + w;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int d = lane * E + e;
      const uint32_t n = (head[codes + slot * (long long)(D / 2) + d / 2] >> (4 * (d & 1))) & 15u;
      o[e] = o[e] * keep + w * fmaf(vp.x, (float)n, vp.y);
    }
    top = m;
  }
#pragma unroll
  for (int e = 0; e < E; e++)
    p.out[t * p.out_stride + (long long)h * D + lane * E + e] = (uint16_t)pack2<BF16>(sum == 0.0f ? 0.0f : o[e] / sum, 0.0f);
  if (p.lse && lane == 0) p.lse[(long long)t * p.q_heads + h] = sum == 0.0f ? -INFINITY : top + logf(sum);
}

}  // namespace
}  // namespace apnn

using namespace apnn;

extern "C" {

size_t apnn_kv4_attention_workspace_bytes(const apnn_kv4_cache* cache, const apnn_kv4_batch* batch, int q_heads) {
  (void)cache;
  (void)batch;
  (void)q_heads;
  return 256;
}

apnn_status apnn_kv4_attention(void* stream, const apnn_kv4_cache* cache, const apnn_kv4_batch* batch,
                               const apnn_kv4_attention_args* a, void* workspace, size_t workspace_bytes) {
  AttentionParams p = {};
  if (!a || a->struct_size != sizeof(apnn_kv4_attention_args) || !a->q || !a->out) return APNN_ERR_INVALID_ARG;
  apnn_status st = kv4_view(cache, &p.cache);
  if (st == APNN_OK) st = kv4_batch(batch, a->rows, &p.batch);
  if (st != APNN_OK) return st;
  if (a->q_heads <= 0 || a->q_heads % cache->heads != 0) return APNN_ERR_INVALID_ARG;
  if ((a->causal != 0 && a->causal != 1) || a->window < 0 || (a->window > 0 && !a->causal)) return APNN_ERR_INVALID_ARG;
  if (!std::isfinite(a->scale)) return APNN_ERR_INVALID_ARG;
  const long long row = (long long)a->q_heads * cache->head_dim;
  if (a->q_stride < row || a->out_stride < row) return APNN_ERR_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) & 15u) != 0 || a->q_stride % 8 != 0 ||
      a->out_stride % 8 != 0 || (reinterpret_cast<uintptr_t>(a->lse) & 3u) != 0 || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
    return APNN_ERR_ALIGNMENT;
  if (!workspace || workspace_bytes < apnn_kv4_attention_workspace_bytes(cache, batch, a->q_heads)) return APNN_ERR_WORKSPACE;
  p.q = static_cast<const uint16_t*>(a->q);
  p.out = static_cast<uint16_t*>(a->out);
  p.lse = a->lse;
  p.q_stride = a->q_stride;
  p.out_stride = a->out_stride;
  p.q_heads = a->q_heads;
  p.group = a->q_heads / cache->heads;
  p.causal = a->causal;
  p.window = a->window;
  p.scale = a->scale;
  void (*const kernels[2][3])(AttentionParams) = {
      {kv4_attention_rows_kernel<false, 64>, kv4_attention_rows_kernel<false, 128>, kv4_attention_rows_kernel<false, 256>},
      {kv4_attention_rows_kernel<true, 64>, kv4_attention_rows_kernel<true, 128>, kv4_attention_rows_kernel<true, 256>}};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(((long long)a->rows * a->q_heads + 3) / 4), 1, 1);
  cfg.blockDim = dim3(128, 1, 1);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  cfg.numAttrs = pdl_attribute(attr);
  cfg.attrs = attr;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernels[cache->type == APNN_TYPE_BF16][cache->head_dim / 128], p);
  return e == cudaSuccess ? APNN_OK : cuda_fail(e, "kv4_attention_rows_kernel");
}

apnn_status apnn_kv4_attention_check(void* stream, const void* workspace) {
  if (!workspace) return APNN_ERR_INVALID_ARG;
  const cudaError_t e = cudaStreamSynchronize(reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? APNN_OK : cuda_fail(e, "apnn_kv4_attention_check");
}

}  // extern "C"
