// Matrix product of 16-bit float activations and weights held as bit planes, with bias, activation and residual in its
// epilogue.
#include <cmath>

#include "linear.cuh"
#include "tc5_common.cuh"

namespace apnn {
namespace {

using namespace tc5;

// ---------------------------------------------------------------------------------------------- few rows
// At most 8 rows of X: the weights are read once and bound it, so nothing of them goes through shared memory.  A warp takes 16
// weight rows, the M operand of mma.sync m16n8k16; the rows of X are its N.  A lane (g, t) reads 16 bytes of each plane of rows
// g and g + 8, 128 elements of K, the four lanes of a row 64 contiguous bytes, a 512-element block ahead.  Which elements of K
// meet in one instruction is free as long as both operands agree, so the fields of a word are taken as they lie, bits b and
// b + 16 side by side: elements 31 - b and 15 - b.  The block pairs its part of X the same way in shared memory, once for its
// eight warps.  K is split over the blocks of a cluster where the weight rows alone are too few warps for the device, and where
// X would not fit; their sums meet in distributed shared memory, added in the order of the ranks.  What bounds it is the spreading,
// some 25 elements a clock and SM at 4 bits (32768 x 16384: 78 us, 3.4 TB/s of planes; 61 at 2 bits, 51 at 1), and below a
// few thousand rows the launch and one chain of loads (4096 x 4096, 4 bits: 6-7 us).
constexpr int FEW_WARPS = 8;
constexpr int FEW_TILE = 16 * FEW_WARPS;      // weight rows of a block
// Rows of X: from nine on linear_tile is as fast (4096 x 4096, 4 bits: 10.9 us against 12.0 with two column tiles here).
constexpr int FEW_ROWS = 8;
constexpr int FEW_SPLIT = 8;                  // largest cluster
constexpr int FEW_X_BYTES = 96 * 1024;        // two blocks to an SM

template <bool BF16>
__device__ __forceinline__ void mma_16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load_stream(const uint32_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Where the pairs 4 c .. 4 c + 3 of word j (of the four that lane t takes of a block) of row m of X lie: 16-byte pieces,
// exchanged so that the lanes of two rows read different banks.
__device__ __forceinline__ int few_x_at(int m, int blocks, int kb, int j, int t, int c) {
  return (((m * blocks + kb) * 4 + j) * 4 + t) * 4 + (c ^ t ^ (m & 1));
}

// four elements of X of which `left` lie before the row's end
__device__ __forceinline__ uint2 few_x_load(const uint16_t* src, int left) {
  if (left >= 4) return __ldg(reinterpret_cast<const uint2*>(src));
  uint2 v = make_uint2(0u, 0u);
  if (left > 0) v.x = src[0];
  if (left > 1) v.x |= (uint32_t)src[1] << 16;
  if (left > 2) v.y = src[2];
  return v;
}

template <int WB, bool BF16>
__global__ void __launch_bounds__(32 * FEW_WARPS, 2) linear_few_rows_kernel(const LinearParams p) {
  using F = Fields<WB>;
  extern __shared__ __align__(64) uint4 x_s[];
  __shared__ float part_s[FEW_TILE][FEW_ROWS + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % p.split;
  const long long n0 = (long long)(blockIdx.x / p.split) * FEW_TILE;
  // this block's 512-element blocks of K
  const int all = (p.kwords + 15) / 16, kb0 = all * rank / p.split, blocks = all * (rank + 1) / p.split - kb0;
  grid_dependency_wait();
  grid_launch_dependents();
  if (p.status_flag && blockIdx.x == 0 && threadIdx.x == 0) *p.status_flag = 0;
  const ZeroPoint<BF16> zero(p.zero);
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};

  // This lane's chunk of the planes for block kb.  Beyond the edges it reads what is there: sums of rows behind N are not
  // stored, and X is zero behind K.
  const uint32_t* base[2];
#pragma unroll
  for (int r = 0; r < 2; r++) base[r] = p.W + min(n0 + warp * 16 + r * 8 + g, (long long)p.N - 1) * p.kwords;
  auto load_weights = [&](int kb, uint4 (&w)[2][WB]) {
    const int word = min((kb0 + min(kb, blocks - 1)) * 16 + t * 4, p.kwords - 4);
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
      for (int b = 0; b < WB; b++) w[r][b] = load_stream(base[r] + b * p.plane_words + word);
  };
  uint4 w0[2][WB], w1[2][WB];
  load_weights(0, w0);

  // X in pieces of four pairs (pair b of a word is elements 31 - b, low half, and 15 - b), zeros behind the row's end; four
  // pieces of a thread in flight at a time
  {
    const int per_row = blocks * 64, total = p.M * per_row;
    int m = 0, at = threadIdx.x;       // row and piece within it
    for (int u = threadIdx.x; u < total; u += 4 * 32 * FEW_WARPS) {
      uint2 hi[4], lo[4];
      int where[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        while (at >= per_row) {
          at -= per_row;
          m++;
        }
        const int word = at >> 2, c = at & 3, k0 = (kb0 * 16 + word) * 32 + 12 - 4 * c;      // elements k0 .. + 3 and k0 + 16 .. + 19
        where[i] = m < p.M ? few_x_at(m, blocks, word >> 4, word & 3, (word >> 2) & 3, c) : -1;
        const uint16_t* src = p.X + m * p.ldx + k0;
        lo[i] = where[i] >= 0 ? few_x_load(src, p.K - k0) : make_uint2(0u, 0u);
        hi[i] = where[i] >= 0 ? few_x_load(src + 16, p.K - k0 - 16) : make_uint2(0u, 0u);
        at += 32 * FEW_WARPS;
      }
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (where[i] >= 0)
          x_s[where[i]] = make_uint4(__byte_perm(hi[i].y, lo[i].y, 0x7632), __byte_perm(hi[i].y, lo[i].y, 0x5410), __byte_perm(hi[i].x, lo[i].x, 0x7632),
                                     __byte_perm(hi[i].x, lo[i].x, 0x5410));
    }
  }
  __syncthreads();

  // lanes behind the last row of X repeat it: their columns are not stored
  const uint4* x_row = x_s + few_x_at(min(g, p.M - 1), blocks, 0, 0, t, 0);
  auto contract = [&](int kb, const uint4 (&w)[2][WB]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      uint32_t f0[F::WORDS], f1[F::WORDS], p0[WB], p1[WB];
#pragma unroll
      for (int b = 0; b < WB; b++) {
        p0[b] = word_of(w[0][b], j);
        p1[b] = word_of(w[1][b], j);
      }
      gather_fields<WB>(p0, f0);
      gather_fields<WB>(p1, f1);
      uint32_t y[16];
#pragma unroll
      for (int c = 0; c < 4; c++) {
        // x_row stands at piece t ^ (m & 1) of its group of four; piece c lies c exchanged bits from there
        const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(x_row + (kb * 4 + j) * 16) ^ (uintptr_t)(c * 16));
        y[4 * c] = v.x;
        y[4 * c + 1] = v.y;
        y[4 * c + 2] = v.z;
        y[4 * c + 3] = v.w;
      }
#pragma unroll
      for (int q = 0; q < F::WORDS; q++)
#pragma unroll
        for (int f = 0; f < F::PER_HALF; f += 2) {
          const int b0 = F::WIDTH * f + q, b1 = F::WIDTH * (f + 1) + q;
          const uint32_t a0 = level_pair<F::WIDTH, BF16>(f0[q], f, zero), a1 = level_pair<F::WIDTH, BF16>(f1[q], f, zero);
          const uint32_t a2 = level_pair<F::WIDTH, BF16>(f0[q], f + 1, zero), a3 = level_pair<F::WIDTH, BF16>(f1[q], f + 1, zero);
          mma_16<BF16>(acc, a0, a1, a2, a3, y[b0], y[b1]);
        }
    }
  };
  for (int kb = 0; kb < blocks; kb += 2) {
    load_weights(kb + 1, w1);
    contract(kb, w0);
    if (kb + 1 == blocks) break;
    load_weights(kb + 2, w0);
    contract(kb + 1, w1);
  }
#pragma unroll
  for (int c = 0; c < 4; c++) part_s[warp * 16 + g + (c >> 1) * 8][2 * t + (c & 1)] = acc[c];
  const int rows = FEW_TILE / p.split;      // of the block's, finished by this rank
  if (p.split > 1) cluster_sync_all();
  else __syncthreads();
  const uint32_t mine = smem_u32(&part_s[0][0]);
  for (int e = threadIdx.x; e < rows * p.M; e += 32 * FEW_WARPS) {
    const int row = rank * rows + e % rows, m = e / rows;
    const long long n = n0 + row;
    if (n >= p.N) continue;
    float sum = 0.0f;
    if (p.split > 1) {
      for (int k = 0; k < p.split; k++) sum += ld_cluster(map_to_cta(mine + (row * (FEW_ROWS + 1) + m) * 4, k));
    } else {
      sum = part_s[row][m];
    }
    store_element<BF16>(p, m, n, sum, __ldg(p.scale + n), p.bias ? __ldg(p.bias + n) : 0.0f);
  }
  if (p.split > 1) cluster_sync_all();      // no rank leaves while another reads its sums
}

template <bool BF16>
void (*few_rows_kernel(int wbits))(LinearParams) {
  return wbits == 1 ? linear_few_rows_kernel<1, BF16> : wbits == 2 ? linear_few_rows_kernel<2, BF16> : wbits == 3 ? linear_few_rows_kernel<3, BF16> : linear_few_rows_kernel<4, BF16>;
}

long long few_x_bytes(int M, int kwords, int split) {
  const int blocks = (kwords + 15) / 16;
  return (long long)M * ((blocks + split - 1) / split) * 1024;
}

// Blocks that share K on the kernel of few rows, 0 where it does not take the call.  The split whose waves (two blocks to an SM) of
// 512-element steps are fewest; beginning and ending a block counts as two steps.  A split is taken as soon as X fits.
int few_rows_split(int M, int N, int kwords) {
  if (M > FEW_ROWS) return 0;
  const int tiles = (N + FEW_TILE - 1) / FEW_TILE, blocks = (kwords + 15) / 16, slots = 2 * device_sm_count();
  int split = 0;
  long long best = -1;
  for (int s = 1; s <= FEW_SPLIT && s <= blocks; s *= 2) {
    const long long steps = ((long long)tiles * s + slots - 1) / slots * ((blocks + s - 1) / s + 2);
    if (few_x_bytes(M, kwords, s) <= FEW_X_BYTES && (best < 0 || steps < best)) {
      best = steps;
      split = s;
    }
  }
  return split;
}

// What the kernels' counts in 32 bits hold: rows of X, rows of all planes and elements of K, up to the ends of the last tile (256 rows)
// and block (512 of K)
bool sizes_held(int M, long long rows, int K) { return M <= 0x7fffffff - 256 && rows <= 0x7fffffff - 256 && K <= 0x7fffffff - 512; }

}  // namespace
}  // namespace apnn

using namespace apnn;

extern "C" apnn_status apnn_linear_planes_plan(int M, int N, int K, int* blocks, int* rows, int* split) {
  if (M <= 0 || N <= 0 || K <= 0 || !blocks || !rows || !split) return APNN_ERR_INVALID_ARG;
  if (!sizes_held(M, N, K)) return APNN_ERR_UNSUPPORTED;
  const int kwords = (K + 127) / 128 * 4;
  LinearPlan plan = {0, FEW_ROWS, few_rows_split(M, N, kwords)};
  if (plan.split == 0) plan = linear_tile_plan(M, N, kwords);
  *blocks = plan.ctas;
  *rows = plan.tn;
  *split = plan.split;
  return APNN_OK;
}

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
  if (!sizes_held(M, (long long)N * wbits, K)) return APNN_ERR_UNSUPPORTED;
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
  p.split = few_rows_split(M, N, p.kwords);
  if (p.split > 0) {
    cudaLaunchConfig_t cfg = {};
    void (*const kernel)(LinearParams) = d->x_type == APNN_TYPE_BF16 ? few_rows_kernel<true>(wbits) : few_rows_kernel<false>(wbits);
    cudaError_t e = ensure_max_smem(reinterpret_cast<const void*>(kernel), FEW_X_BYTES);
    if (e != cudaSuccess) return cuda_fail(e, "linear_few_rows_kernel shared memory");
    cfg.gridDim = dim3((unsigned)((N + FEW_TILE - 1) / FEW_TILE * p.split), 1, 1);
    cfg.blockDim = dim3(32 * FEW_WARPS, 1, 1);
    cfg.dynamicSmemBytes = (size_t)few_x_bytes(M, p.kwords, p.split);
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    cfg.numAttrs = pdl_attribute(attr);
    if (p.split > 1) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
      attr[cfg.numAttrs].val.clusterDim.x = (unsigned)p.split;
      attr[cfg.numAttrs].val.clusterDim.y = 1;
      attr[cfg.numAttrs].val.clusterDim.z = 1;
      cfg.numAttrs++;
    }
    cfg.attrs = attr;
    e = cudaLaunchKernelEx(&cfg, kernel, p);
    return e == cudaSuccess ? APNN_OK : cuda_fail(e, "linear_few_rows_kernel");
  }
  return linear_tile(reinterpret_cast<cudaStream_t>(stream), p, d->x_type == APNN_TYPE_BF16);
}
