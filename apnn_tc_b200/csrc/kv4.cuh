// The 4-bit key / value cache: device view, batch geometry and 16-bit float conversions shared by its kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "api_internal.h"

namespace apnn {

struct Kv4View {
  uint8_t* data;
  long long page_stride;   // bytes
  int pages, heads, page_size, page_shift;
  long long head_bytes;    // page_size * (D + 8)
};
struct Kv4Batch {
  const int* cu_q;
  const int* kv_len;
  const int* table;
  long long table_stride;
  int sequences, table_width, max_q, rows;
};

constexpr int MOST_HEADS = 1 << 20;      // of keys, of queries: what a row's pieces are counted in

// Checks shared by the entry points; fill the kernels' views.
apnn_status kv4_view(const apnn_kv4_cache* c, Kv4View* v);
apnn_status kv4_batch(const apnn_kv4_batch* b, int rows, Kv4Batch* out);

// Two 16-bit floats of a word as fp32, and back (round to nearest even).
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool BF16>
__device__ __forceinline__ float round16(float x) {
  return BF16 ? __bfloat162float(__float2bfloat16_rn(x)) : __half2float(__float2half_rn(x));
}

// The sequence of row t (a whole warp asks): the last b with cu_q[b] <= t, -1 behind the last row.  128 entries a round, all of
// a round's loads and the row count's at once, so up to 128 sequences cost one load's latency.
__device__ __forceinline__ int sequence_of(const int* cu_q, int sequences, int t, int lane) {
  const int end = __ldg(cu_q + sequences);
  int lo = 0, n = sequences;   // the answer lies in [lo, lo + n)
  do {
    const int step = (n + 127) >> 7;
    int at[4], hits = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int k = (lane + 32 * i) * step;
      at[i] = k < n ? __ldg(cu_q + lo + k) : 0x7fffffff;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) hits += __popc(__ballot_sync(0xffffffffu, at[i] <= t));
    const int hit = max(hits - 1, 0);
    lo += hit * step;
    n = min(step, n - hit * step);
  } while (n > 1);
  return t >= end ? -1 : lo;
}

// Byte address of head 0 of the page that holds `pos` of sequence b, or null where there is none.
__device__ __forceinline__ uint8_t* page_of(const Kv4View& c, const Kv4Batch& g, int b, int pos) {
  if (pos < 0) return nullptr;
  const int slot = pos >> c.page_shift;
  if (slot >= g.table_width) return nullptr;
  const int page = __ldg(g.table + b * g.table_stride + slot);
  if (page < 0 || page >= c.pages) return nullptr;
  return c.data + page * c.page_stride;
}

}  // namespace apnn
