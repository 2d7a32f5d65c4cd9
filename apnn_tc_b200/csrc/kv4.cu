// The 4-bit key / value cache: keys and values of new rows into its pages, together with the norm of each query and key
// head and the rotation by position, and rows back out as values.
#include "kv4.cuh"
#include "tc5_common.cuh"

namespace apnn {

apnn_status kv4_view(const apnn_kv4_cache* c, Kv4View* v) {
  if (!c || c->struct_size != sizeof(apnn_kv4_cache) || !c->data) return APNN_ERR_INVALID_ARG;
  if (c->type != APNN_TYPE_BF16 && c->type != APNN_TYPE_FP16) return APNN_ERR_INVALID_ARG;
  if (c->pages <= 0 || c->heads <= 0) return APNN_ERR_INVALID_ARG;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return APNN_ERR_UNSUPPORTED;
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

constexpr int APPEND_THREADS = 256;

// A block takes one row of the batch; D / 8 lanes take one head of it, eight elements each (one 16-byte load, one word of
// levels), so the reductions over a head are shuffles and the rotation's partner sits in another lane of the group.
template <bool BF16, int D>
__global__ void __launch_bounds__(APPEND_THREADS) kv4_append_kernel(const AppendParams p) {
  constexpr int LANES = D / 8;
  constexpr int PER_BLOCK = APPEND_THREADS / LANES;
  const int t = blockIdx.x;
  const int lane = threadIdx.x & 31;
  const int c = lane % LANES;                     // which eight elements of the head
  const int total = p.q_heads + 2 * p.kv_heads;
  grid_dependency_wait();
  const int b = sequence_of(p.batch.cu_q, p.batch.sequences, t, lane);
  if (b < 0) return;                              // a row behind the last sequence
  const int first = __ldg(p.batch.cu_q + b);
  const int pos = __ldg(p.batch.kv_len + b) - (__ldg(p.batch.cu_q + b + 1) - first) + (t - first);
  uint8_t* page = page_of(p.cache, p.batch, b, pos);
  const int slot = pos & (p.cache.page_size - 1);
  for (int r0 = 0; r0 < total; r0 += PER_BLOCK) {
    const int r = r0 + threadIdx.x / LANES;
    const bool live = r < total;
    const int kind = !live || r >= p.q_heads + p.kv_heads ? 2 : r >= p.q_heads ? 1 : 0;   // q, k or v
    const int h = r - (kind == 0 ? 0 : kind == 1 ? p.q_heads : p.q_heads + p.kv_heads);
    float y[8];
    if (live) {
      const uint4 w = *reinterpret_cast<const uint4*>(p.in[kind] + (long long)t * p.stride[kind] + (long long)h * D + c * 8);
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float2 f = unpack2<BF16>(words[i]);
        y[2 * i] = f.x;
        y[2 * i + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) y[i] = 0.0f;
    }
    const uint16_t* weight = kind == 2 ? nullptr : p.norm[kind];
    if (p.norm[0] != nullptr || p.norm[1] != nullptr) {     // uniform: the shuffles below take every lane
      // squares of 16-bit floats are exact in fp32; their sum is held in fp64, so its order does not show in the levels
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < 8; i++) sum += (double)__fmul_rn(y[i], y[i]);
#pragma unroll
      for (int d = 1; d < LANES; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (weight != nullptr) {
        const float scale = __fdiv_rn(1.0f, __fsqrt_rn((float)(sum / D + p.eps)));
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(weight + c * 8));
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float2 f = unpack2<BF16>(words[i]);
          y[2 * i] = __fmul_rn(__fmul_rn(y[2 * i], scale), f.x);
          y[2 * i + 1] = __fmul_rn(__fmul_rn(y[2 * i + 1], scale), f.y);
        }
      }
    }
    if (p.rotary_dim > 0) {
      const int half = p.rotary_dim / 2;
      const bool turned = kind != 2 && c * 8 < p.rotary_dim;
      const bool known = pos >= 0 && pos < p.rotary_rows;
      const float* row = p.rotary + (long long)(known ? pos : 0) * p.rotary_dim;
      if (p.interleaved) {
        if (turned) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float cs = __ldg(row + c * 4 + i), sn = __ldg(row + half + c * 4 + i);
            const float a = y[2 * i], d = y[2 * i + 1];
            y[2 * i] = __fsub_rn(__fmul_rn(a, cs), __fmul_rn(d, sn));
            y[2 * i + 1] = __fadd_rn(__fmul_rn(d, cs), __fmul_rn(a, sn));
          }
        }
      } else {
        const bool upper = c * 8 >= half;
        const int partner = (lane - c) + (turned ? (upper ? c - half / 8 : c + half / 8) : c);
        const int at = c * 8 - (upper ? half : 0);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float other = __shfl_sync(0xffffffffu, y[i], partner);
          if (turned) {
            const float cs = __ldg(row + at + i), sn = __ldg(row + half + at + i);
            y[i] = upper ? __fadd_rn(__fmul_rn(y[i], cs), __fmul_rn(other, sn)) : __fsub_rn(__fmul_rn(y[i], cs), __fmul_rn(other, sn));
          }
        }
      }
      if (kind != 2 && !known) {
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = __int_as_float(0x7fc00000);
      }
    }
    if (live && kind == 0) {
      uint4 o;
      o.x = pack2<BF16>(y[0], y[1]);
      o.y = pack2<BF16>(y[2], y[3]);
      o.z = pack2<BF16>(y[4], y[5]);
      o.w = pack2<BF16>(y[6], y[7]);
      *reinterpret_cast<uint4*>(p.q_out + (long long)t * p.q_out_stride + (long long)h * D + c * 8) = o;
    }
    float lo = y[0], hi = y[0], all = __fmul_rn(y[0], 0.0f);    // all: 0, or NaN once an element is not finite
#pragma unroll
    for (int i = 1; i < 8; i++) {
      lo = fminf(lo, y[i]);
      hi = fmaxf(hi, y[i]);
      all = __fadd_rn(all, __fmul_rn(y[i], 0.0f));
    }
#pragma unroll
    for (int d = 1; d < LANES; d *= 2) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
      all += __shfl_xor_sync(0xffffffffu, all, d);
    }
    if (live && kind != 0 && page != nullptr) {
      float step = round16<BF16>(__fsub_rn(__fdiv_rn(hi, 15.0f), __fdiv_rn(lo, 15.0f)));
      float low = round16<BF16>(lo);
      if (step < 1.17549435e-38f) step = 0.0f;
      uint32_t word = 0;
      if (all != 0.0f || !isfinite(step) || !isfinite(low)) {     // NaN compares unequal
        step = low = __int_as_float(0x7fc00000);
      } else if (step > 0.0f) {
        const float inverse = __fdiv_rn(1.0f, step);
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float level = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(y[i], low), inverse)), 0.0f), 15.0f);
          word |= (uint32_t)(int)level << (4 * i);
        }
      }
      uint8_t* head = page + h * p.cache.head_bytes;
      const int part = kind - 1;    // keys, values
      const long long codes = (long long)p.cache.page_size * (D / 2);
      *reinterpret_cast<uint32_t*>(head + part * codes + (long long)slot * (D / 2) + c * 4) = word;
      if (c == 0) *reinterpret_cast<uint32_t*>(head + 2 * codes + (part * p.cache.page_size + slot) * 4ll) = pack2<BF16>(step, low);
    }
  }
}

template <bool BF16, int D>
__global__ void __launch_bounds__(APPEND_THREADS) kv4_read_kernel(const Kv4View cache, const Kv4Batch batch, uint16_t* k_out, uint16_t* v_out) {
  constexpr int LANES = D / 8;
  constexpr int PER_BLOCK = APPEND_THREADS / LANES;
  const int t = blockIdx.x;
  const int lane = threadIdx.x & 31;
  const int c = lane % LANES;
  grid_dependency_wait();
  const int b = sequence_of(batch.cu_q, batch.sequences, t, lane);
  if (b < 0) return;
  const int first = __ldg(batch.cu_q + b);
  const int pos = __ldg(batch.kv_len + b) - (__ldg(batch.cu_q + b + 1) - first) + (t - first);
  const uint8_t* page = page_of(cache, batch, b, pos);
  const int slot = pos & (cache.page_size - 1);
  const long long codes = (long long)cache.page_size * (D / 2);
  for (int r = threadIdx.x / LANES; r < 2 * cache.heads; r += PER_BLOCK) {
    const int part = r >= cache.heads ? 1 : 0;
    const int h = r - part * cache.heads;
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
      // step * level is exact in fp32 (at most 15 bits), so the sum is the only rounding before the store's
      const float e = __fmaf_rn(par.x, (float)((word >> (8 * i)) & 15u), par.y);
      const float f = __fmaf_rn(par.x, (float)((word >> (8 * i + 4)) & 15u), par.y);
      o[i] = pack2<BF16>(e, f);
    }
    *reinterpret_cast<uint4*>((part ? v_out : k_out) + ((long long)t * cache.heads + h) * D + c * 8) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

template <typename... Params, typename... Args>
apnn_status launch_rows(const char* what, void (*kernel)(Params...), int rows, void* stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows, 1, 1);
  cfg.blockDim = dim3(APPEND_THREADS, 1, 1);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  cfg.numAttrs = pdl_attribute(attr);
  cfg.attrs = attr;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  return e == cudaSuccess ? APNN_OK : cuda_fail(e, what);
}

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
  if (a->rotary_dim % 16 != 0) return APNN_ERR_UNSUPPORTED;
  if (a->rotary_dim > 0 && (!a->rotary || a->rotary_rows <= 0)) return APNN_ERR_INVALID_ARG;
  if (!(a->eps >= 0.0) || !(a->eps < 1e30)) return APNN_ERR_INVALID_ARG;
  const long long row = (long long)cache->heads * D;
  if (a->k_stride < row || a->v_stride < row) return APNN_ERR_INVALID_ARG;
  if (a->q && (a->q_stride < (long long)a->q_heads * D || a->q_out_stride < (long long)a->q_heads * D)) return APNN_ERR_INVALID_ARG;
  if (off16(a->k) || off16(a->v) || off16(a->q) || off16(a->q_out) || off16(a->q_norm) || off16(a->k_norm) ||
      (reinterpret_cast<uintptr_t>(a->rotary) & 3u) != 0)
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
  void (*const kernels[2][3])(AppendParams) = {{kv4_append_kernel<false, 64>, kv4_append_kernel<false, 128>, kv4_append_kernel<false, 256>},
                                               {kv4_append_kernel<true, 64>, kv4_append_kernel<true, 128>, kv4_append_kernel<true, 256>}};
  return launch_rows("kv4_append_kernel", kernels[cache->type == APNN_TYPE_BF16][D / 128], a->rows, stream, p);
}

apnn_status apnn_kv4_read(void* stream, const apnn_kv4_cache* cache, const apnn_kv4_batch* batch, void* k_out, void* v_out, int rows) {
  Kv4View view = {};
  Kv4Batch geo = {};
  if (!k_out || !v_out) return APNN_ERR_INVALID_ARG;
  apnn_status st = kv4_view(cache, &view);
  if (st == APNN_OK) st = kv4_batch(batch, rows, &geo);
  if (st != APNN_OK) return st;
  if (off16(k_out) || off16(v_out)) return APNN_ERR_ALIGNMENT;
  void (*const kernels[2][3])(Kv4View, Kv4Batch, uint16_t*, uint16_t*) = {{kv4_read_kernel<false, 64>, kv4_read_kernel<false, 128>, kv4_read_kernel<false, 256>},
                                                                          {kv4_read_kernel<true, 64>, kv4_read_kernel<true, 128>, kv4_read_kernel<true, 256>}};
  return launch_rows("kv4_read_kernel", kernels[cache->type == APNN_TYPE_BF16][cache->head_dim / 128], rows, stream, view, geo,
                     static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out));
}

}  // extern "C"
