// Attention over the 4-bit cache: what its kernels share.
#pragma once
#include <cmath>

#include "kv4.cuh"
#include "tc5_common.cuh"

namespace apnn {

struct AttentionParams {
  Kv4View cache;
  Kv4Batch batch;
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  long long q_stride, out_stride;
  int q_heads, group, causal, window;
  float scale;
  int* status_flag;
};

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Weights of the values carry the values' steps and are rounded to fp16, so what the largest step leaves of a smaller one counts.  Up
// to this many powers of two between the steps met, all rows of a block share one power of two for them: a row that sees only the
// smallest steps then keeps fp16's eleven bits down to weights of 2^-10 of its reference point.  Steps further apart (a row that is
// masked or all but weightless may hold any) take a path on which each row has its own.
constexpr int STEP_SPAN = 10;
// Whether steps lie too far apart: 2^top is above the largest, `under` the fp32 bits of the smallest (not 0), less 1; all ones: none.
__device__ __forceinline__ bool steps_far_apart(int top, uint32_t under) {
  return under != 0xffffffffu && top + 126 - (int)((under + 1u) >> 23) > STEP_SPAN;
}

// Two fp32 in one instruction.
struct Pair { unsigned long long v; };
__device__ __forceinline__ Pair pair(float x, float y) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(x), "f"(y));
  return p;
}
__device__ __forceinline__ float2 unpair(Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
  return f;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}

// Four elements of an output row from their sums: row r of the sequence's rows for key head h.
template <bool BF16, int D, typename S>
__device__ __forceinline__ void finish_row(const AttentionParams& p, const S& s, int h, int r, int d, float M, float L, float4 v) {
  const int i = r / p.group, head = h * p.group + (r - i * p.group);
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;      // no key: 0; NaN stays NaN
  const long long t = s.first + i;
  *reinterpret_cast<uint2*>(p.out + t * p.out_stride + (long long)head * D + d) = make_uint2(pack2<BF16>(v.x * inv, v.y * inv), pack2<BF16>(v.z * inv, v.w * inv));
  if (d == 0 && p.lse != nullptr) p.lse[t * p.q_heads + head] = L == 0.0f ? -INFINITY : M * LN2 + logf(L);
}

// One sequence of the call: which rows, which keys any of them sees.
struct Span {
  int first, n;        // rows first .. first + n - 1
  int pos0;            // position of the first
  int len;             // keys there are
  int begin, end;      // keys that some row sees lie in [begin, end)
  int tile0, tiles;    // tiles of `TILE` keys over them; one (empty) tile where there is no key, none without rows
};
template <int TILE>
__device__ __forceinline__ Span span_of(const AttentionParams& p, int b) {
  Span s;
  s.first = __ldg(p.batch.cu_q + b);
  const int all = __ldg(p.batch.cu_q + b + 1) - s.first;
  s.n = s.first < 0 ? 0 : min(min(all, p.batch.max_q), p.batch.rows - s.first);
  const int kv = __ldg(p.batch.kv_len + b);
  s.pos0 = kv - all;
  s.len = (int)min((long long)kv, (long long)p.batch.table_width << p.cache.page_shift);
  s.begin = 0;
  s.end = s.len;
  if (p.causal) {
    s.end = min(s.end, s.pos0 + s.n);
    if (p.window > 0) s.begin = max(0, s.pos0 + 1 - p.window);
  }
  s.tile0 = s.begin / TILE;
  s.tiles = s.n <= 0 ? 0 : s.end > s.begin ? (s.end + TILE - 1) / TILE - s.tile0 : 1;
  return s;
}

// More rows of a sequence than the flow kernel takes (kv4_prompt.cu).
size_t kv4_prompt_workspace_bytes(const apnn_kv4_cache* cache, const apnn_kv4_batch* batch, int group);
apnn_status kv4_prompt(cudaStream_t s, const apnn_kv4_cache* cache, const apnn_kv4_batch* batch, const AttentionParams& p, void* workspace);

}  // namespace apnn
