// The 4-bit key / value cache: keys and values of new rows into its pages, together with the norm of each query and key
// head and the rotation by position, and rows back out as values.
#include <algorithm>

#include "kv4.cuh"
#include "tc5_common.cuh"

namespace apnn {

apnn_status kv4_view(const apnn_kv4_cache* c, Kv4View* v) {
  if (!c || c->struct_size != sizeof(apnn_kv4_cache) || !c->data) return APNN_ERR_INVALID_ARG;
  if (c->type != APNN_TYPE_BF16 && c->type != APNN_TYPE_FP16) return APNN_ERR_INVALID_ARG;
  if (c->pages <= 0 || c->heads <= 0) return APNN_ERR_INVALID_ARG;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return APNN_ERR_UNSUPPORTED;
  if (c->heads > MOST_HEADS) return APNN_ERR_UNSUPPORTED;
  if (c->page_size < 8 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)) != 0) return APNN_ERR_UNSUPPORTED;
  v->head_bytes = (long long)c->page_size * (c->head_dim + 8);
  if ((reinterpret_cast<uintptr_t>(c->data) & 15u) != 0 || c->page_stride % 16 != 0) return APNN_ERR_ALIGNMENT;
  if (c->page_stride < v->head_bytes * c->heads) return APNN_ERR_INVALID_ARG;
  v->data = static_cast<uint8_t*>(c->data);
  v->page_stride = c->page_stride;
  v->pages = c->pages;
  v->heads = c->heads;
  v->page_size = c->page_size;
  v->page_shift = __builtin_ctz((unsigned)c->page_size);
  return APNN_OK;
}

apnn_status kv4_batch(const apnn_kv4_batch* b, int rows, Kv4Batch* out) {
  if (!b || b->struct_size != sizeof(apnn_kv4_batch) || !b->cu_q || !b->kv_len || !b->table) return APNN_ERR_INVALID_ARG;
  if (b->sequences <= 0 || b->table_width <= 0 || b->max_q <= 0 || rows <= 0) return APNN_ERR_INVALID_ARG;
  if (b->table_stride < b->table_width) return APNN_ERR_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(b->cu_q) | reinterpret_cast<uintptr_t>(b->kv_len) | reinterpret_cast<uintptr_t>(b->table)) & 3u) != 0)
    return APNN_ERR_ALIGNMENT;
  out->cu_q = b->cu_q;
  out->kv_len = b->kv_len;
  out->table = b->table;
  out->table_stride = b->table_stride;
  out->sequences = b->sequences;
  out->table_width = b->table_width;
  out->max_q = b->max_q;
  out->rows = rows;
  return APNN_OK;
}

namespace {

using namespace tc5;

struct AppendParams {
  Kv4View cache;
  Kv4Batch batch;
  const uint16_t* in[3];      // q, k, v
  long long stride[3];
  uint16_t* q_out;
  long long q_out_stride;
  int q_heads, kv_heads;
  const uint16_t* norm[2];    // of q, of k
  double eps;
  int rotary_dim, interleaved, rotary_rows;
  const float* rotary;
};

// Warps of a block: as few passes over a row's heads as eight warps allow, in equal parts (12 pieces of a row: two passes of
// six warps).
constexpr int ROW_WARPS = 8;
// Warps that fit a multiprocessor with the registers that the launch bounds leave.
constexpr int APPEND_RESIDENT = 32, READ_RESIDENT = 48;

constexpr float FIFTEENTH = 1.0f / 15.0f;

// max that keeps NaN, so that one NaN among a row's elements shows in its step
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Where the rows t0 .. t0 + R - 1 of the batch lie, lane i holding row t0 + i; R <= 32.
struct Places {
  int count;               // rows before the last sequence's end and the tensors'
  int pos;
  uint8_t* page;           // null where there is none
};
__device__ __forceinline__ Places places_of(const Kv4View& cache, const Kv4Batch& batch, int t0, int R, int lane) {
  Places out = {min(R, min(__ldg(batch.cu_q + batch.sequences), batch.rows) - t0), 0, nullptr};
  if (out.count <= 0) return out;
  int b = sequence_of(batch.cu_q, batch.sequences, t0, lane);
  const int t = t0 + min(lane, out.count - 1);
  int next = __ldg(batch.cu_q + b + 1);
  if (t >= next) {         // a later sequence than t0's: the last one that begins at t or before
    int n = batch.sequences - b;
    while (n > 1) {
      const int up = n >> 1;
      const bool reached = __ldg(batch.cu_q + b + up) <= t;
      b += reached ? up : 0;
      n = reached ? n - up : up;
    }
    next = __ldg(batch.cu_q + b + 1);
  }
  out.pos = __ldg(batch.kv_len + b) - next + t;      // the sequence's rows are its last
  out.page = page_of(cache, batch, b, out.pos);
  return out;
}

// D / 8 lanes take one head of a row, eight elements each (one 16-byte load, one word of levels), so the reductions over a
// head are shuffles and the rotation's partner sits in another lane of the group.  A warp's heads are all queries, all keys
// or all values, so a query is not quantised and a value neither normed nor turned.  A block takes `R` rows: finding a row's
// sequence, position and page is a chain of four dependent loads, paid once for all of them (lane i looks for row i) and not
// for each (measured with a row a block: 42 us for 9325 rows of 3 * 16 heads of 64, all of it that chain).  Inputs are loaded
// one row ahead, the first while the chain runs.  At that size 200 instructions for each 32 * 8 elements bound it: they issue in
// 69% of the cycles.  Packed arithmetic saved a tenth of them and cost the registers that keep 32 warps resident (35 us against 33).
template <bool BF16, int D>
__global__ void __launch_bounds__(ROW_WARPS * 32, APPEND_RESIDENT / ROW_WARPS) kv4_append_kernel(const AppendParams p, const int R) {
  constexpr int LANES = D / 8;
  constexpr int HEADS = 32 / LANES;               // of a warp
  const int t0 = blockIdx.x * R;
  const int lane = threadIdx.x & 31;
  const int c = lane % LANES;                     // which eight elements of the head
  const int of_q = (p.q_heads + HEADS - 1) / HEADS, of_k = (p.kv_heads + HEADS - 1) / HEADS;
  const int pieces = of_q + 2 * of_k;
  grid_dependency_wait();
  int w = threadIdx.x >> 5, kind = 0, h = -1, r = 0;
  const uint16_t* source = nullptr;
  const auto begin = [&]() {                      // piece w, from its first row
    kind = w >= of_q + of_k ? 2 : w >= of_q ? 1 : 0;          // q, k or v
    h = (w - (kind == 0 ? 0 : kind == 1 ? of_q : of_q + of_k)) * HEADS + lane / LANES;
    if (w >= pieces || h >= (kind == 0 ? p.q_heads : p.kv_heads)) h = -1;
    source = p.in[kind] + (long long)t0 * p.stride[kind] + (long long)h * D + c * 8;
  };
  const auto fetch = [&]() { return h >= 0 ? *reinterpret_cast<const uint4*>(source) : make_uint4(0, 0, 0, 0); };
  begin();
  uint4 in = fetch();
  const Places at = places_of(p.cache, p.batch, t0, R, lane);
  if (at.count <= 0) return;                      // rows behind the last sequence
  const long long codes = (long long)p.cache.page_size * (D / 2);
  const int half = p.rotary_dim / 2;
  const bool turned = c * 8 < p.rotary_dim;
  const bool upper = c * 8 >= half;
  const int partner = (lane - c) + (turned ? (upper ? c - half / 8 : c + half / 8) : c);

  while (w < pieces) {
    const int kind_now = kind, h_now = h, t = t0 + r;
    const bool live = h >= 0;
    const uint32_t words[4] = {in.x, in.y, in.z, in.w};
    const int pos = __shfl_sync(0xffffffffu, at.pos, r);
    uint8_t* page = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(at.page), r));
    if (++r < at.count) {
      source += p.stride[kind];
    } else {
      r = 0;
      w += blockDim.x >> 5;
      begin();
    }
    in = fetch();
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = unpack2<BF16>(words[i]);
      y[2 * i] = f.x;
      y[2 * i + 1] = f.y;
    }
    if (kind_now != 2) {
      const bool known = p.rotary_dim == 0 || (pos >= 0 && pos < p.rotary_rows);
      float cs[8], sn[8];
      if (turned) {
        const float* row = p.rotary + (long long)(known ? pos : 0) * p.rotary_dim + (p.interleaved ? c * 4 : c * 8 - (upper ? half : 0));
#pragma unroll
        for (int i = 0; i < 2; i++) {
          if (i == 1 && p.interleaved) break;
          const float4 x = __ldg(reinterpret_cast<const float4*>(row) + i), y = __ldg(reinterpret_cast<const float4*>(row + half) + i);
          cs[4 * i] = x.x, cs[4 * i + 1] = x.y, cs[4 * i + 2] = x.z, cs[4 * i + 3] = x.w;
          sn[4 * i] = y.x, sn[4 * i + 1] = y.y, sn[4 * i + 2] = y.z, sn[4 * i + 3] = y.w;
        }
      }
      const uint16_t* weight = p.norm[kind_now];
      if (weight != nullptr) {
        // Squares are taken in fp64, where those of 16-bit floats are exact (in fp32 those of bf16 leave its range from 2^64 on and
        // lose bits below 2^-63); so is their sum, so that its order does not show in the levels
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < 8; i++) sum = fma((double)y[i], (double)y[i], sum);
#pragma unroll
        for (int d = 1; d < LANES; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const float scale = __fdiv_rn(1.0f, __fsqrt_rn((float)(sum / D + p.eps)));
        const uint4 g = __ldg(reinterpret_cast<const uint4*>(weight + c * 8));
        const uint32_t gains[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float2 f = unpack2<BF16>(gains[i]);
          y[2 * i] = __fmul_rn(__fmul_rn(y[2 * i], scale), f.x);
          y[2 * i + 1] = __fmul_rn(__fmul_rn(y[2 * i + 1], scale), f.y);
        }
      }
      if (p.rotary_dim > 0) {
        if (p.interleaved) {
          if (turned) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const float a = y[2 * i], d = y[2 * i + 1];
              y[2 * i] = __fsub_rn(__fmul_rn(a, cs[i]), __fmul_rn(d, sn[i]));
              y[2 * i + 1] = __fadd_rn(__fmul_rn(d, cs[i]), __fmul_rn(a, sn[i]));
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float other = __shfl_sync(0xffffffffu, y[i], partner);
            if (turned) y[i] = __fadd_rn(__fmul_rn(y[i], cs[i]), __fmul_rn(other, upper ? sn[i] : -sn[i]));      // a c - b s, b c + a s
          }
        }
        if (!known) {
#pragma unroll
          for (int i = 0; i < 8; i++) y[i] = __int_as_float(0x7fc00000);
        }
      }
    }
    if (kind_now == 0) {
      if (live) {
        uint4 o;
        o.x = pack2<BF16>(y[0], y[1]);
        o.y = pack2<BF16>(y[2], y[3]);
        o.z = pack2<BF16>(y[4], y[5]);
        o.w = pack2<BF16>(y[6], y[7]);
        *reinterpret_cast<uint4*>(p.q_out + (long long)t * p.q_out_stride + (long long)h_now * D + c * 8) = o;
      }
      continue;
    }
    float lo = y[0], hi = y[0];
#pragma unroll
    for (int i = 1; i < 8; i++) {
      lo = fminf(lo, y[i]);
      hi = max_nan(hi, y[i]);
    }
#pragma unroll
    for (int d = 1; d < LANES; d *= 2) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, d));
    }
    if (live && page != nullptr) {
      // an infinity among the elements is lo or hi, a NaN is hi: either way the step is not finite
      float step = round16<BF16>(__fsub_rn(__fmul_rn(hi, FIFTEENTH), __fmul_rn(lo, FIFTEENTH)));
      float low = round16<BF16>(lo);
      if (step < 1.17549435e-38f) step = 0.0f;
      uint32_t word = 0;
      if (!isfinite(step) || !isfinite(low)) {
        step = low = __int_as_float(0x7fc00000);
      } else if (step > 0.0f) {
        const float inverse = __fdiv_rn(1.0f, step);
        // adding 2^23 rounds to the nearest even integer and leaves it in the low bits; eight of them joined by shifted sums,
        // less the same sum of 2^23's own bits, 0x4b000000 * (1 + 16)
        word = 0u - 0xfb000000u;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float level = fminf(fmaxf(__fmul_rn(__fsub_rn(y[i], low), inverse), 0.0f), 15.0f);
          word += __float_as_uint(__fadd_rn(level, 8388608.0f)) << (4 * i);
        }
      }
      uint8_t* head = page + h_now * p.cache.head_bytes;
      const int part = kind_now - 1;    // keys, values
      const int slot = pos & (p.cache.page_size - 1);
      *reinterpret_cast<uint32_t*>(head + part * codes + (long long)slot * (D / 2) + c * 4) = word;
      if (c == 0) *reinterpret_cast<uint32_t*>(head + 2 * codes + (part * p.cache.page_size + slot) * 4ll) = pack2<BF16>(step, low);
    }
  }
}

// The same split of a row's heads; keys in the first half of the pieces, values in the second.
template <bool BF16, int D>
__global__ void __launch_bounds__(ROW_WARPS * 32, READ_RESIDENT / ROW_WARPS) kv4_read_kernel(const Kv4View cache, const Kv4Batch batch,
                                                                                               uint16_t* k_out, uint16_t* v_out, const int R) {
  constexpr int LANES = D / 8;
  constexpr int HEADS = 32 / LANES;
  const int t0 = blockIdx.x * R;
  const int lane = threadIdx.x & 31;
  const int c = lane % LANES;
  const int of_k = (cache.heads + HEADS - 1) / HEADS;
  grid_dependency_wait();
  const Places at = places_of(cache, batch, t0, R, lane);
  if (at.count <= 0) return;
  const long long codes = (long long)cache.page_size * (D / 2);
  for (int w = threadIdx.x >> 5; w < 2 * of_k; w += blockDim.x >> 5) {
    const int part = w >= of_k ? 1 : 0;
    const int h = (w - part * of_k) * HEADS + lane / LANES;
#pragma unroll 4
    for (int r = 0; r < at.count; r++) {
      const int slot = __shfl_sync(0xffffffffu, at.pos, r) & (cache.page_size - 1);
      const uint8_t* page = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(at.page), r));
      if (h >= cache.heads) continue;
      float2 par = make_float2(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
      uint32_t word = 0;
      if (page != nullptr) {
        const uint8_t* head = page + h * cache.head_bytes;
        word = *reinterpret_cast<const uint32_t*>(head + part * codes + (long long)slot * (D / 2) + c * 4);
        par = unpack2<BF16>(*reinterpret_cast<const uint32_t*>(head + 2 * codes + (part * cache.page_size + slot) * 4ll));
      }
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        // a level in the low bits of 2^23 is 2^23 plus the level: conversions to float run at an eighth of this.
        // step * level is exact in fp32 (at most 15 bits), so the sum is the only rounding before the store's
        const float e = __uint_as_float(((word >> (8 * i)) & 15u) | 0x4b000000u) - 8388608.0f;
        const float f = __uint_as_float(((word >> (8 * i + 4)) & 15u) | 0x4b000000u) - 8388608.0f;
        o[i] = pack2<BF16>(__fmaf_rn(par.x, e, par.y), __fmaf_rn(par.x, f, par.y));
      }
      *reinterpret_cast<uint4*>((part ? v_out : k_out) + ((long long)(t0 + r) * cache.heads + h) * D + c * 8) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

template <typename... Params, typename... Args>
apnn_status launch_rows(const char* what, void (*kernel)(Params...), int rows, int pieces, int resident, void* stream, Args... args) {
  // rows of a block: what one wave of resident blocks leaves to each, up to the lanes that look them up (9325 rows of 3 * 16
  // heads of 64, append and read: a row a block 42 + 20 us, 8 rows 34 + 11, this rule 31 + 11; from a cold L2 40 + 19)
  const int passes = (pieces + ROW_WARPS - 1) / ROW_WARPS, warps = (pieces + passes - 1) / passes;
  const int wave = device_sm_count() * (resident / warps);
  const int R = std::min((rows + wave - 1) / wave, 32);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((rows + R - 1) / R), 1, 1);
  cfg.blockDim = dim3((unsigned)warps * 32u, 1, 1);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  cfg.numAttrs = pdl_attribute(attr);
  cfg.attrs = attr;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args..., R);
  return e == cudaSuccess ? APNN_OK : cuda_fail(e, what);
}

// Warps' worth of heads, at 32 / (D / 8) heads a warp.
int pieces_of(int heads, int D) { return (heads * (D / 8) + 31) / 32; }

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

}  // namespace
}  // namespace apnn

using namespace apnn;

extern "C" {

apnn_status apnn_kv4_append(void* stream, const apnn_kv4_cache* cache, const apnn_kv4_batch* batch, const apnn_kv4_append_args* a) {
  AppendParams p = {};
  if (!a || a->struct_size != sizeof(apnn_kv4_append_args) || !a->k || !a->v) return APNN_ERR_INVALID_ARG;
  apnn_status st = kv4_view(cache, &p.cache);
  if (st == APNN_OK) st = kv4_batch(batch, a->rows, &p.batch);
  if (st != APNN_OK) return st;
  const int D = cache->head_dim;
  if ((a->q != nullptr) != (a->q_out != nullptr) || (a->q && a->q_heads <= 0)) return APNN_ERR_INVALID_ARG;
  if (a->rotary_dim < 0 || a->rotary_dim > D || (a->interleaved != 0 && a->interleaved != 1)) return APNN_ERR_INVALID_ARG;
  if (a->rotary_dim % 16 != 0 || (a->q && a->q_heads > MOST_HEADS)) return APNN_ERR_UNSUPPORTED;
  if (a->rotary_dim > 0 && (!a->rotary || a->rotary_rows <= 0)) return APNN_ERR_INVALID_ARG;
  if (!(a->eps >= 0.0) || !(a->eps < 1e30)) return APNN_ERR_INVALID_ARG;
  const long long row = (long long)cache->heads * D;
  if (a->k_stride < row || a->v_stride < row) return APNN_ERR_INVALID_ARG;
  if (a->q && (a->q_stride < (long long)a->q_heads * D || a->q_out_stride < (long long)a->q_heads * D)) return APNN_ERR_INVALID_ARG;
  if (off16(a->k) || off16(a->v) || off16(a->q) || off16(a->q_out) || off16(a->q_norm) || off16(a->k_norm) ||
      off16(a->rotary))
    return APNN_ERR_ALIGNMENT;
  if (a->k_stride % 8 != 0 || a->v_stride % 8 != 0 || (a->q && (a->q_stride % 8 != 0 || a->q_out_stride % 8 != 0))) return APNN_ERR_ALIGNMENT;
  p.in[0] = static_cast<const uint16_t*>(a->q);
  p.in[1] = static_cast<const uint16_t*>(a->k);
  p.in[2] = static_cast<const uint16_t*>(a->v);
  p.stride[0] = a->q_stride;
  p.stride[1] = a->k_stride;
  p.stride[2] = a->v_stride;
  p.q_out = static_cast<uint16_t*>(a->q_out);
  p.q_out_stride = a->q_out_stride;
  p.q_heads = a->q ? a->q_heads : 0;
  p.kv_heads = cache->heads;
  p.norm[0] = static_cast<const uint16_t*>(a->q_norm);
  p.norm[1] = static_cast<const uint16_t*>(a->k_norm);
  p.eps = a->eps;
  p.rotary_dim = a->rotary_dim;
  p.interleaved = a->interleaved;
  p.rotary_rows = a->rotary_rows;
  p.rotary = a->rotary;
  void (*const kernels[2][3])(AppendParams, int) = {{kv4_append_kernel<false, 64>, kv4_append_kernel<false, 128>, kv4_append_kernel<false, 256>},
                                               {kv4_append_kernel<true, 64>, kv4_append_kernel<true, 128>, kv4_append_kernel<true, 256>}};
  return launch_rows("kv4_append_kernel", kernels[cache->type == APNN_TYPE_BF16][D / 128], a->rows,
                     pieces_of(p.q_heads, D) + 2 * pieces_of(cache->heads, D), APPEND_RESIDENT, stream, p);
}

apnn_status apnn_kv4_read(void* stream, const apnn_kv4_cache* cache, const apnn_kv4_batch* batch, void* k_out, void* v_out, int rows) {
  Kv4View view = {};
  Kv4Batch geo = {};
  if (!k_out || !v_out) return APNN_ERR_INVALID_ARG;
  apnn_status st = kv4_view(cache, &view);
  if (st == APNN_OK) st = kv4_batch(batch, rows, &geo);
  if (st != APNN_OK) return st;
  if (off16(k_out) || off16(v_out)) return APNN_ERR_ALIGNMENT;
  void (*const kernels[2][3])(Kv4View, Kv4Batch, uint16_t*, uint16_t*, int) = {
      {kv4_read_kernel<false, 64>, kv4_read_kernel<false, 128>, kv4_read_kernel<false, 256>},
      {kv4_read_kernel<true, 64>, kv4_read_kernel<true, 128>, kv4_read_kernel<true, 256>}};
  return launch_rows("kv4_read_kernel", kernels[cache->type == APNN_TYPE_BF16][cache->head_dim / 128], rows,
                     2 * pieces_of(cache->heads, cache->head_dim), READ_RESIDENT, stream, view, geo,
                     static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out));
}

}  // extern "C"
