// Attention over the 4-bit cache.
#include <type_traits>

#include "kv4_attention.cuh"

namespace apnn {
namespace {

using namespace tc5;

// D(16x8, fp32) += A(16x16, fp16) * B(16x8, fp16)
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// transpose of an 8x8 block of 16-bit elements, two per lane
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
template <int WORDS>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t* r) {
  if (WORDS == 1) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r[0]) : "r"(a));
  if (WORDS == 2) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(a));
  if (WORDS == 4) asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}

// ---------------------------------------------------------------------------------------------- single and few tokens
// The rows of a sequence that share a key head (its queries times the group, at most 8 NQ) stand against tiles of 128 keys,
// 32 for each of four warps, which run on their own until the end of a segment.  Scores are computed transposed: a tile of
// 16 keys is the M operand of mma.sync m16n8k16 and the query rows its N, so eight rows fill the instruction and every key
// is spread from its nibbles once.  A word of eight levels becomes fp16 operand pairs by masking alone:
//   w & 0x000f000f, w & 0x00f000f0, (w >> 8) & 0x000f000f, (w >> 8) & 0x00f000f0
// are pairs of fp16 subnormals, n 2^-24 and n 2^-20, which the tensor core multiplies exactly; the queries stand in the
// matching order, those at the second and fourth mask divided by 16, scaled by a power of two to fp16's range (exact).
//   s_j = scale (step_j sum_d q_d n_jd + low_j sum_d q_d)
// The weights of the values carry the values' step, w_j = 2^(s_j - m) step_j 2^(6 - R) with 2^R above every step seen and m
// at most 8 below the largest s (so at most 2^14, 2^15 at the end of the range; fp16's eleven bits hold down to 2^-20 of the
// reference point); they are rounded once, and
//   sum_j p_j v_jd = 2^(R - 6) (sum_j w_j n_jd - 8 sum_j w_j) + sum_j p_j (low_j + 8 step_j)
// takes the same rounded w in both sums, so the rounding meets levels centred at 8, not 0..15 (half the error of fp16
// results).  Where the steps of a segment lie more than 2^STEP_SPAN apart, the rest of it goes with a reference point of each row for the
// values, apart from that of the softmax: w_j = 2^(s_j - m + log2 step_j - a) with a at most 14 below the largest exponent.
// Value words of two keys are put side by side by PRMT to give pairs along the keys.
// HBM is the floor, (D + 8) bytes per key and head; the steady state is bound by instruction issue (some 600 for 32 keys of a
// warp, half of the cycles, the integer pipe at 46%), and about 10 us go to the start, the meeting of the warps and the joining
// kernel (64 sequences of up to 16384 keys, 212 MB: 60 us, 3.5 TB/s; one of 65536, 71 MB: 25 us in a row on the device, 27 with the
// host's call).  Looking after the steps' range costs one comparison a tile; 64 sequences of 4096 keys whose steps lie far apart take
// 93 us, others 77.
constexpr int FLOW_WARPS = 4;
constexpr int FLOW_KEYS = 32;                       // per warp and tile
constexpr int FLOW_TILE = FLOW_WARPS * FLOW_KEYS;   // 128
constexpr int FLOW_STAGES = 3;
// What beginning and ending a (sequence, head) costs, in tiles, when work is shared out (64 ragged sequences of 8 heads: 69 us
// at 1, 62 at 2, 63 at 3 and 4).
constexpr int FLOW_SEGMENT = 2;
constexpr int UNSPLIT_KEYS = 512;   // tables of at most this many positions: no split, no second launch

template <int D, int NQ>
struct Flow {
  static constexpr int WK = D / 32;    // words of a key row per lane (four lanes hold a row)
  static constexpr int WV = D / 64;    // words of a value row per lane (eight lanes)
  static constexpr int ROW = D / 2, ROW_LOG = D == 64 ? 5 : D == 128 ? 6 : 7;
  static constexpr int V_AT = FLOW_KEYS * ROW, KP_AT = 2 * V_AT, VP_AT = KP_AT + FLOW_KEYS * 4;
  static constexpr int STAGE = VP_AT + FLOW_KEYS * 4;
  static constexpr int RING = FLOW_STAGES * STAGE;
  static constexpr int ROWS = 8 * NQ;
  static constexpr int MERGE = ROWS * (D + 4) * 4;       // a warp's part of the exchange at a segment's end: o, then m and l
  static constexpr int PER_WARP = RING > MERGE ? RING : MERGE;
  static constexpr bool Q_IN_REGS = NQ * WK <= 4;
  static constexpr int Q_BYTES = Q_IN_REGS ? 0 : 2 * WK * NQ * 32 * 8;
  static constexpr int SMEM = FLOW_WARPS * PER_WARP + Q_BYTES + ROWS * 8 + 128;
  // per SM (one row, D = 128, on the device: one sequence of 65536 keys 24.3 us at 2, 24.5 at 3, 26.0 at 4; 64 ragged ones 67, 60, 60)
  static constexpr int BLOCKS = NQ <= 2 && D != 256 ? 3 : 2;
  static constexpr int SLOT = ROWS * (D + 2);            // floats of a partial result
};

// The key of row r of an MMA operand, within eight: keys 2 t of the four lanes that read different value rows at once then lie
// in different banks (D = 64; two by two at D = 128), while eight lanes that read key rows still take whole 128-byte lines.
__device__ __forceinline__ int flow_key(int r) { return r ^ ((r >> 1) & 1) ^ ((r >> 2) & 1); }

__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ const uint8_t* shuffle_ptr(const uint8_t* p, int lane) {
  return reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(p), lane));
}

struct FlowParams {
  AttentionParams a;
  int2* pieces;     // [sequences * heads]: first block and number of the partial results of a (sequence, head), 0: none
  float* slots;     // [2 * blocks][Flow::SLOT]
  int split;
  int run_shift;    // log2 of the keys of a tile's 32 that lie in one page: 3, 4 or 5
};

template <bool BF16, int D, int NQ>
__global__ void __launch_bounds__(32 * FLOW_WARPS, Flow<D, NQ>::BLOCKS) kv4_attention_flow_kernel(const FlowParams fp) {
  using F = Flow<D, NQ>;
  const AttentionParams& p = fp.a;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  uint8_t* my_smem = smem + warp * F::PER_WARP;
  const uint32_t ring = smem_u32(my_smem);
  uint2* q_s = reinterpret_cast<uint2*>(smem + FLOW_WARPS * F::PER_WARP);
  float2* qf_s = reinterpret_cast<float2*>(smem + FLOW_WARPS * F::PER_WARP + F::Q_BYTES);   // per row: factor of the products, of the lows
  int* scan_s = reinterpret_cast<int*>(smem + FLOW_WARPS * F::PER_WARP + F::Q_BYTES + F::ROWS * 8);
  const int heads = p.cache.heads, sequences = p.batch.sequences;
  grid_dependency_wait();
  grid_launch_dependents();   // the joining kernel waits for this whole grid anyway
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.status_flag = 0;

  // ---- which units this block takes: an equal share of all, in order.  A (sequence, head) is FLOW_SEGMENT units of overhead,
  // then a unit for each tile.
  int u0, u1, b = 0, h = 0, loc = 0;
  int share = 0, longer = 0;     // units of a block; the first `longer` blocks have one more
  Span s;
  auto weight = [&](const Span& x) { return x.tiles == 0 ? 0 : (x.tiles + FLOW_SEGMENT) * heads; };
  if (fp.split) {
    // false for a block without a share.  No share between two is empty: the joining kernel counts on it
    auto take = [&](int total) {
      const int sharing = min(total, (int)gridDim.x), block = (int)blockIdx.x;
      if (block >= sharing) return false;
      share = total / sharing;
      longer = total - share * sharing;
      u0 = share * block + min(block, longer);
      u1 = u0 + share + (block < longer ? 1 : 0);
      return true;
    };
    const bool at_once = sequences <= 32 * FLOW_WARPS;
    if (!at_once) {
      int sum = 0;
      for (int i = threadIdx.x; i < sequences; i += 32 * FLOW_WARPS) sum += weight(span_of<FLOW_TILE>(p, i));
      sum = __reduce_add_sync(0xffffffffu, sum);
      if (lane == 0) scan_s[warp] = sum;
      __syncthreads();
      if (!take(scan_s[0] + scan_s[1] + scan_s[2] + scan_s[3])) return;
    }
    // the sequence of unit u0, 128 sequences at a time
    int before = 0;
    for (int base = 0;; base += 32 * FLOW_WARPS) {
      if (base > 0) __syncthreads();
      const int i = base + threadIdx.x;
      const int mine = i < sequences ? weight(span_of<FLOW_TILE>(p, i)) : 0;
      int inc = mine;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += o;
      }
      if (lane == 31) scan_s[4 + warp] = inc;
      __syncthreads();
      int at = before;
      for (int w = 0; w < warp; w++) at += scan_s[4 + w];
      before += scan_s[4] + scan_s[5] + scan_s[6] + scan_s[7];
      if (at_once && !take(before)) return;
      if (u0 >= at + inc - mine && u0 < at + inc) {
        scan_s[8] = i;
        scan_s[9] = at + inc - mine;
      }
      if (before > u0) break;     // uniform; the total is more than u0, so a sequence is found
    }
    __syncthreads();
    b = scan_s[8];
    s = span_of<FLOW_TILE>(p, b);
    h = (u0 - scan_s[9]) / (s.tiles + FLOW_SEGMENT);
    loc = (u0 - scan_s[9]) - h * (s.tiles + FLOW_SEGMENT);
  } else {
    // a block takes a (sequence, head) whole
    u0 = blockIdx.x;
    u1 = sequences * heads;
  }

  for (int u = u0; u < u1;) {
    int t0 = 0, nt, bh_unit = 0;
    if (fp.split) {
      while (s.tiles == 0 || h == heads) {     // on to the next sequence with rows
        h = 0;
        s = span_of<FLOW_TILE>(p, ++b);
      }
      bh_unit = u - loc;
      t0 = max(loc - FLOW_SEGMENT, 0);
      nt = min(s.tiles, u1 - bh_unit - FLOW_SEGMENT) - t0;
    } else {
      b = u / heads;
      h = u - b * heads;
      s = span_of<FLOW_TILE>(p, b);
      nt = s.tiles;
    }
    const int next_u = fp.split ? bh_unit + s.tiles + FLOW_SEGMENT : u + gridDim.x;
    if (nt <= 0) {      // only overhead units lie in this share, or a sequence without rows
      u = next_u;
      loc = 0;
      if (fp.split) h++;
      continue;
    }
    const int rows = s.n * p.group;     // at most 8 NQ

    // ---- copies of this warp's 32-key pieces of the segment, 16 bytes a lane: key levels, value levels and the parameters of
    // both lie in runs of 8 to 32 keys of one page.  Four lanes look up the page of a run, a tile ahead.  (Bulk copies of a run by a
    // lane each: they leave a warp one at a time, 1000 clk for a tile's four, half as long as its attention.)
    const int key0 = (s.tile0 + t0) * FLOW_TILE + warp * FLOW_KEYS;
    const int run_shift = fp.run_shift, run_log = F::ROW_LOG + run_shift, v_off = p.cache.page_size * F::ROW;
    const uint8_t* head_base = p.cache.data + h * p.cache.head_bytes;
    const int* trow = p.batch.table + (long long)b * p.batch.table_stride;
    const uint32_t all_live = 0xffffu >> (16 - 4 * (FLOW_KEYS >> run_shift));
    const uint32_t lane_dst = ring + lane * 16;
    // this lane's run of the next tile to look up, and where the looking ends (end <= table_width * page_size: within the table)
    int at_key = key0 + ((lane >> 2) << run_shift);
    const int stop = (lane >> 2) < (FLOW_KEYS >> run_shift) ? min(s.end, key0 + nt * FLOW_TILE) : 0;
    auto source = [&]() -> const uint8_t* {      // the first key's levels; a page of more than 32 keys holds the tile in one run
      const uint8_t* src = nullptr;
      if (at_key < stop) {
        const int id = __ldg(trow + (at_key >> p.cache.page_shift));
        if ((uint32_t)id < (uint32_t)p.cache.pages) src = head_base + id * p.cache.page_stride + (at_key & (p.cache.page_size - 1)) * F::ROW;
      }
      at_key += FLOW_TILE;
      return src;
    };
    // returns which runs there are, four bits for each
    auto issue = [&](int i, const uint8_t* src) -> uint32_t {
      uint32_t live = 0;
      if (i < nt) {
        live = __ballot_sync(0xffffffffu, src != nullptr);
        const uint32_t dst = lane_dst + (i % FLOW_STAGES) * F::STAGE;
        const int first = (key0 + i * FLOW_TILE) & (p.cache.page_size - 1);
        // from a run's key levels to the keys' parameters (the page holds both parts' levels first)
        const int params = 2 * v_off - (run_shift == 5 ? first * (F::ROW - 4) : 0);
        if (run_shift == 5) {
          const uint8_t* from = shuffle_ptr(src, 0);
          if (live != 0) {
            const uint8_t *k = from + lane * 16, *v = k + v_off;
#pragma unroll
            for (int c = 0; c < F::V_AT / 512; c++) {
              copy16(dst + c * 512, k + c * 512);
              copy16(dst + F::V_AT + c * 512, v + c * 512);
            }
            if (lane < 16) copy16(dst + F::KP_AT, from + params + (lane >> 3) * (4 * p.cache.page_size) + (lane & 7) * 16);
          }
        } else {
#pragma unroll
          for (int c = 0; c < F::V_AT / 512; c++) {
            const int byte = c * 512 + lane * 16;
            const uint8_t* from = shuffle_ptr(src, (byte >> run_log) * 4);
            if (from != nullptr) {
              from += byte & ((1 << run_log) - 1);
              copy16(dst + c * 512, from);
              copy16(dst + F::V_AT + c * 512, from + v_off);
            }
          }
          const int byte = (lane & 7) * 16;
          const uint8_t* from = shuffle_ptr(src, (byte >> (2 + run_shift)) * 4);
          if (from != nullptr && lane < 16)
            copy16(dst + F::KP_AT, from + params + (lane >> 3) * (4 * p.cache.page_size) + (byte & ((4 << run_shift) - 1)));
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      return live;
    };
    const uint8_t* src = source();
    uint32_t live_of[FLOW_STAGES - 1];      // of the tiles on their way
#pragma unroll
    for (int i = 0; i < FLOW_STAGES - 1; i++) {
      const uint8_t* next = source();
      live_of[i] = issue(i, src);
      src = next;
    }

    // ---- the queries as fp16 operands, while the first keys are on their way.  A group of four lanes (t) shares a row.
    uint32_t qr[F::Q_IN_REGS ? 2 * F::WK * NQ * 2 : 1];
    auto load_row = [&](int r, uint2* frags) {       // this lane's 8 WK elements of row r -> 2 WK operand pairs; factors to shared memory
      float x[8 * F::WK];
      const bool live = r < rows;
      const int i = live ? r / p.group : 0;
      const uint16_t* src = p.q + (long long)(s.first + i) * p.q_stride + (long long)(h * p.group + (live ? r - i * p.group : 0)) * D;
#pragma unroll
      for (int w = 0; w < F::WK; w++) {
        // word w of this lane's key words: element 32 t + 8 w (D = 128), 16 t + 8 w (64), 128 (w / 4) + 32 t + 8 (w % 4) (256)
        const int d = D == 64 ? 16 * t + 8 * w : 128 * (w / 4) + 32 * t + 8 * (w & 3);
        const uint4 v = live ? *reinterpret_cast<const uint4*>(src + d) : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float2 f = unpack2<BF16>(vv[j]);
          x[8 * w + 2 * j] = f.x;
          x[8 * w + 2 * j + 1] = f.y;
        }
      }
      float top = 0.0f, sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8 * F::WK; j++) {
        top = fmaxf(top, fabsf(x[j]));
        sum += x[j];
      }
#pragma unroll
      for (int d = 1; d < 4; d *= 2) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        sum += __shfl_xor_sync(0xffffffffu, sum, d);
      }
      // power of two that takes the row's largest element to [2^14, 2^15); rows of zeros and of infinities as they are
      const int e = (int)(__float_as_uint(top) >> 23) - 127;
      const int shift = top > 0.0f && e < 128 ? 14 - max(e, -100) : 0;
      const float up = __uint_as_float((uint32_t)(127 + shift) << 23);
      if (t == 0) qf_s[r] = make_float2(p.scale * LOG2E * __uint_as_float((uint32_t)(127 - shift) << 23), p.scale * LOG2E * sum);
#pragma unroll
      for (int w = 0; w < F::WK; w++) {
        const float* y = x + 8 * w;
        const float down = up * 0.0625f;
        frags[2 * w] = make_uint2(pack2<false>(y[0] * up, y[4] * up), pack2<false>(y[1] * down, y[5] * down));
        frags[2 * w + 1] = make_uint2(pack2<false>(y[2] * up, y[6] * up), pack2<false>(y[3] * down, y[7] * down));
      }
    };
    if (F::Q_IN_REGS) {
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        uint2 frags[2 * F::WK];
        load_row(q * 8 + g, frags);     // every warp writes the same factors
#pragma unroll
        for (int k = 0; k < 2 * F::WK; k++) {
          qr[(k * NQ + q) * 2] = frags[k].x;
          qr[(k * NQ + q) * 2 + 1] = frags[k].y;
        }
      }
    } else {
      for (int q = warp; q < NQ; q += FLOW_WARPS) {
        uint2 frags[2 * F::WK];
        load_row(q * 8 + g, frags);
#pragma unroll
        for (int k = 0; k < 2 * F::WK; k++) q_s[(k * NQ + q) * 32 + lane] = frags[k];
      }
    }
    __syncthreads();
    Pair qf[NQ], ql[NQ];
#pragma unroll
    for (int q = 0; q < NQ; q++) {
      const float2 f0 = qf_s[q * 8 + 2 * t], f1 = qf_s[q * 8 + 2 * t + 1];
      qf[q] = pair(f0.x, f1.x);
      ql[q] = pair(f0.y, f1.y);
    }
    // the keys every row sees: no mask is looked at there
    const int last_begin = p.causal && p.window > 0 ? max(0, s.pos0 + s.n - p.window) : 0;
    const int first_end = p.causal ? min(s.len, s.pos0 + 1) : s.len;

    float o[F::WV][4][NQ][4];
    Pair l[NQ], vsum[NQ];
#pragma unroll
    for (int q = 0; q < NQ; q++)
#pragma unroll
      for (int c = 0; c < 4; c++) {
#pragma unroll
        for (int w = 0; w < F::WV; w++)
#pragma unroll
          for (int j = 0; j < 4; j++) o[w][j][q][c] = 0.0f;
      }
#pragma unroll
    for (int q = 0; q < NQ; q++) l[q] = vsum[q] = pair(0.0f, 0.0f);
    const int fk = flow_key(g), fv = flow_key(2 * t);
    // reference points, negated (0 where no key was met), and 8 above them; 2^R is above every value step met so far, within
    // fp32's range; lift = 2^(6 - R)
    Pair below[NQ];
    float rise_at[2 * NQ];
#pragma unroll
    for (int q = 0; q < NQ; q++) below[q] = pair(0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < 2 * NQ; c++) rise_at[c] = -INFINITY;
    auto reference = [&](int c) {
      const float2 f = unpair(below[c >> 1]);
      return rise_at[c] == -INFINITY ? -INFINITY : c & 1 ? -f.y : -f.x;
    };
    int R = -112;
    uint32_t step_bits = 0;     // the fp32 bits of 2^R, 0 before the first key: larger steps raise R
    uint32_t under = 0xffffffffu;      // the bits of a power of two no step but 0 was below, less 1; all ones before the first
    float lift = __uint_as_float((uint32_t)(127 + 6 + 112) << 23);
    float apart[2 * NQ];        // steps far apart: the values' reference points less the softmax's, log2

    // False, with nothing done, where the steps turn out to lie too far apart for one power of two

    auto attend = [&](auto tag, auto far_tag, int key, uint32_t at, uint32_t live) -> bool {
      constexpr bool WHOLE = decltype(tag)::value;      // every row sees every key: no mask is looked at
      constexpr bool FAR = decltype(far_tag)::value;
      // ---- scores of two tiles of 16 keys
      float sc[2][NQ][4];
#pragma unroll
      for (int mt = 0; mt < 2; mt++)
#pragma unroll
        for (int q = 0; q < NQ; q++)
#pragma unroll
          for (int c = 0; c < 4; c++) sc[mt][q][c] = 0.0f;
      constexpr int WL = F::WK < 4 ? F::WK : 4;     // words of one load
#pragma unroll
      for (int w0 = 0; w0 < F::WK; w0 += WL) {
        uint32_t kw[2][2][WL];
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
          for (int hi = 0; hi < 2; hi++) {
            // w0 is 0 or, at D = 256, 4: bytes 16 t or 64 + 16 t
            lds_words<WL>(at + (mt * 16 + hi * 8) * F::ROW + fk * F::ROW + 4 * WL * t + 16 * w0, kw[mt][hi]);
          }
#pragma unroll
        for (int w = 0; w < WL; w++) {
#pragma unroll
          for (int half = 0; half < 2; half++) {
            const int k = 2 * (w0 + w) + half;
            uint2 bq[NQ];
#pragma unroll
            for (int q = 0; q < NQ; q++)
              bq[q] = F::Q_IN_REGS ? make_uint2(qr[(k * NQ + q) * 2], qr[(k * NQ + q) * 2 + 1]) : q_s[(k * NQ + q) * 32 + lane];
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
              const uint32_t x = half ? kw[mt][0][w] >> 8 : kw[mt][0][w], y = half ? kw[mt][1][w] >> 8 : kw[mt][1][w];
#pragma unroll
              for (int q = 0; q < NQ; q++)
                mma_f16(sc[mt][q], x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u, bq[q].x, bq[q].y);
            }
          }
        }
      }
      // ---- the rows' parameters; scores in the log2 domain; running maximum
      float2 kp[4], vp[4];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        kp[r] = unpack2<BF16>(lds32(at + F::KP_AT + r * 32 + fk * 4));
        kp[r].x *= 16777216.0f;      // the levels are multiples of 2^-24
        vp[r] = unpack2<BF16>(lds32(at + F::VP_AT + r * 32 + fk * 4));
      }
      uint32_t seen[2 * NQ];     // bit r: the key of parameter r is visible to the row of column c
      if (!WHOLE) {
#pragma unroll
        for (int c = 0; c < 2 * NQ; c++) {
          const int r = (c >> 1) * 8 + 2 * t + (c & 1);
          const int pos = s.pos0 + min(r / p.group, s.n - 1);
          const int end = p.causal ? min(s.len, pos + 1) : s.len;
          const int begin = p.causal && p.window > 0 ? pos + 1 - p.window : 0;
          seen[c] = 0;
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const int j = key + k * 8 + fk;
            if (j < end && j >= begin && ((live >> (((k * 8) >> fp.run_shift) * 4)) & 1u)) seen[c] |= 1u << k;
          }
        }
      }
      float top[2 * NQ];
#pragma unroll
      for (int c = 0; c < 2 * NQ; c++) top[c] = -INFINITY;
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int q = 0; q < NQ; q++) {
          float* x = sc[r >> 1][q] + 2 * (r & 1);
          const float2 v = unpair(fma2(mul2(pair(x[0], x[1]), pair(kp[r].x, kp[r].x)), qf[q], mul2(pair(kp[r].y, kp[r].y), ql[q])));
          x[0] = WHOLE || ((seen[2 * q] >> r) & 1u) ? v.x : -INFINITY;
          x[1] = WHOLE || ((seen[2 * q + 1] >> r) & 1u) ? v.y : -INFINITY;
          top[2 * q] = fmaxf(top[2 * q], x[0]);
          top[2 * q + 1] = fmaxf(top[2 * q + 1], x[1]);
        }
      // exponents of the largest and the smallest value step of these keys (a step that is not finite shows in its weight instead)
      uint32_t bits = 0;
      if (!FAR) {
        bits = __float_as_uint(fabsf(unpack2<BF16>(lds32(at + F::VP_AT + lane * 4)).x));
        if (bits >= 0x7f800000u || (!WHOLE && (key + lane >= s.end || key + lane < s.begin || !((live >> ((lane >> fp.run_shift) * 4)) & 1u)))) bits = 0;
      }
      // The reference point m follows the running maximum only where that has risen by more than 2^8: weights then stay below
      // 2^8 of it, and most tiles after a segment's first neither exchange maxima nor touch the sums.
      bool moved = !FAR && (bits > step_bits || bits - 1u < under);
#pragma unroll
      for (int c = 0; c < 2 * NQ; c++) moved |= top[c] > rise_at[c];
      if (__any_sync(0xffffffffu, moved)) {
        float shrink = 1.0f;      // 2^(R - rise)
        if (!FAR) {
          const int rise = max(R, min((int)(__reduce_max_sync(0xffffffffu, bits) >> 23) - 126, 127));
          const uint32_t least = min(under, __reduce_min_sync(0xffffffffu, bits - 1u));
          if (steps_far_apart(rise, least)) return false;
          if (least != 0xffffffffu) under = max((least + 1u) & 0x7f800000u, 1u) - 1u;
          shrink = __uint_as_float((uint32_t)max(127 + R - rise, 0) << 23);
          R = rise;
          step_bits = (uint32_t)(127 + R) << 23;
          lift = __uint_as_float((uint32_t)(127 + 6 - R) << 23);
        }
        float kept[2 * NQ];
#pragma unroll
        for (int c = 0; c < 2 * NQ; c++) {
#pragma unroll
          for (int d = 4; d < 32; d *= 2) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], d));
          const float m = reference(c);
          top[c] = fmaxf(top[c], m);
          const float keep = m == top[c] ? 1.0f : ex2(m - top[c]);       // -inf - x: 0
          rise_at[c] = top[c] + 8.0f;
          const float k = keep * shrink;
          kept[c] = keep;
          if (FAR) {
            if (m != top[c]) apart[c] += m - top[c];      // the values' own point stays; -inf where no key was met
          } else {
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
              for (int w = 0; w < F::WV; w++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[w][j][c >> 1][(c & 1) + 2 * e] *= k;
            }
          }
        }
#pragma unroll
        for (int q = 0; q < NQ; q++) {
          l[q] = mul2(l[q], pair(kept[2 * q], kept[2 * q + 1]));
          vsum[q] = mul2(vsum[q], pair(kept[2 * q], kept[2 * q + 1]));
          below[q] = pair(top[2 * q] == -INFINITY ? 0.0f : -top[2 * q], top[2 * q + 1] == -INFINITY ? 0.0f : -top[2 * q + 1]);
        }
      }
      float lg[4];      // log2 of the value steps, to 2^-22 of themselves or of 1: far below an fp16 rounding of the weights
      if (FAR) {
        float most[2 * NQ];
#pragma unroll
        for (int c = 0; c < 2 * NQ; c++) most[c] = -INFINITY;
        bool over = false;
#pragma unroll
        for (int r = 0; r < 4; r++) lg[r] = __log2f(fabsf(vp[r].x));
#pragma unroll
        for (int c = 0; c < 2 * NQ; c++) {
          const float2 f = unpair(below[c >> 1]);
#pragma unroll
          for (int r = 0; r < 4; r++) most[c] = fmaxf(most[c], sc[r >> 1][c >> 1][2 * (r & 1) + (c & 1)] + (c & 1 ? f.y : f.x) + lg[r]);      // NaN counts as none
          over |= most[c] > apart[c] + 14.0f;
        }
        if (__any_sync(0xffffffffu, over)) {
#pragma unroll
          for (int c = 0; c < 2 * NQ; c++) {
#pragma unroll
            for (int d = 4; d < 32; d *= 2) most[c] = fmaxf(most[c], __shfl_xor_sync(0xffffffffu, most[c], d));
            const float up = fmaxf(apart[c], most[c] - 6.0f), k = up == apart[c] ? 1.0f : ex2(apart[c] - up);
            apart[c] = up;
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
              for (int w = 0; w < F::WV; w++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[w][j][c >> 1][(c & 1) + 2 * e] *= k;
            }
          }
        }
      }
      // ---- weights, and their products with the values.  Levels are centred at 8 tile by tile: sums of what is all positive
      // grow far above the result, and the tensor cores truncate (3000 keys, fp16: 4.2e-4 off with one subtraction at the end, so
      // 2.8e-4, which the roundings of the weights and of the result make up)
      float eights[NQ][4];
#pragma unroll
      for (int q = 0; q < NQ; q++)
#pragma unroll
        for (int c = 0; c < 4; c++) eights[q][c] = 0.0f;
      uint32_t wt[2][NQ][2];
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float step = vp[r].x * lift, mid = fmaf(8.0f, vp[r].x, vp[r].y);
#pragma unroll
        for (int q = 0; q < NQ; q++) {
          const float* x = sc[r >> 1][q] + 2 * (r & 1);
          const float2 z = unpair(add2(pair(x[0], x[1]), below[q]));
          const Pair e = pair(ex2(z.x), ex2(z.y));
          l[q] = add2(l[q], e);
          float2 w;
          if (FAR) {
            w.x = copysignf(ex2(z.x + (lg[r] - (apart[2 * q] == -INFINITY ? 0.0f : apart[2 * q]))), vp[r].x);
            w.y = copysignf(ex2(z.y + (lg[r] - (apart[2 * q + 1] == -INFINITY ? 0.0f : apart[2 * q + 1]))), vp[r].x);
          } else {
            w = unpair(mul2(e, pair(step, step)));
          }
          if (WHOLE) {
            vsum[q] = fma2(e, pair(mid, mid), vsum[q]);
          } else {      // a masked place may hold NaN
            const bool on0 = (seen[2 * q] >> r) & 1u, on1 = (seen[2 * q + 1] >> r) & 1u;
            w.x = on0 ? w.x : 0.0f;
            w.y = on1 ? w.y : 0.0f;
            vsum[q] = fma2(e, pair(on0 ? mid : 0.0f, on1 ? mid : 0.0f), vsum[q]);
          }
          wt[r >> 1][q][r & 1] = transpose8x8(pack2<false>(w.x, w.y));
        }
      }
#pragma unroll
      for (int mt = 0; mt < 2; mt++) {
        uint32_t vw[4][F::WV];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          lds_words<F::WV>(at + F::V_AT + (mt * 16 + (k >> 1) * 8) * F::ROW + (fv ^ (k & 1)) * F::ROW + 4 * F::WV * g, vw[k]);
        }
#pragma unroll
        for (int q = 0; q < NQ; q++) mma_f16(eights[q], 0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u, wt[mt][q][0], wt[mt][q][1]);
#pragma unroll
        for (int w = 0; w < F::WV; w++) {
#pragma unroll
          for (int j = 0; j < 4; j++) {
            uint32_t x = __byte_perm(vw[0][w], vw[1][w], j < 2 ? 0x5410 : 0x7632);
            uint32_t y = __byte_perm(vw[2][w], vw[3][w], j < 2 ? 0x5410 : 0x7632);
            if (j & 1) {
              x >>= 8;
              y >>= 8;
            }
#pragma unroll
            for (int q = 0; q < NQ; q++)
              mma_f16(o[w][j][q], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, wt[mt][q][0], wt[mt][q][1]);
          }
        }
      }
#pragma unroll
      for (int q = 0; q < NQ; q++) {
        const Pair down = pair(-eights[q][0], -eights[q][1]), down16 = mul2(down, pair(16.0f, 16.0f));
#pragma unroll
        for (int w = 0; w < F::WV; w++)
#pragma unroll
          for (int j = 0; j < 4; j++) {      // the second row of a word's pair stands 16 times too high
            const float2 a = unpair(add2(pair(o[w][j][q][0], o[w][j][q][1]), down)), b = unpair(add2(pair(o[w][j][q][2], o[w][j][q][3]), down16));
            o[w][j][q][0] = a.x;
            o[w][j][q][1] = a.y;
            o[w][j][q][2] = b.x;
            o[w][j][q][3] = b.y;
          }
      }
      return true;
    };

    int i = 0;
    auto walk = [&](auto far_tag) {      // from tile i on, to the end or to a tile whose steps lie too far apart
      for (; i < nt; i++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(FLOW_STAGES - 2) : "memory");
        __syncwarp();
        const uint32_t live = live_of[0];
        const int key = key0 + i * FLOW_TILE;
        if (key < s.end && key + FLOW_KEYS > s.begin) {       // warp-uniform
          const uint32_t at = ring + (i % FLOW_STAGES) * F::STAGE;
          bool done;
          if (!decltype(far_tag)::value && live == all_live && key >= last_begin && key + FLOW_KEYS <= first_end) done = attend(std::true_type(), std::false_type(), key, at, live);
          else done = attend(std::false_type(), far_tag, key, at, live);
          if (!done) return;
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < FLOW_STAGES - 2; k++) live_of[k] = live_of[k + 1];
        live_of[FLOW_STAGES - 2] = issue(i + FLOW_STAGES - 1, src);
        src = source();
      }
    };
    walk(std::false_type());
    const bool far = i < nt;      // of this warp
    if (far) {
#pragma unroll
      for (int c = 0; c < 2 * NQ; c++) apart[c] = rise_at[c] == -INFINITY ? -INFINITY : (float)(R - 6);
      walk(std::true_type());
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();

    // ---- the four warps' results meet in shared memory
    {
      float* mine = reinterpret_cast<float*>(my_smem);
      constexpr float LEVEL = 16777216.0f;      // the levels are multiples of 2^-24
#pragma unroll
      for (int c = 0; c < 2 * NQ; c++) {
        const int r = (c >> 1) * 8 + 2 * t + (c & 1);
        // the values' reference point in two factors: 2^(R - 6), R >= -112
        const float root = ex2(0.5f * apart[c]);
        const float unit = LEVEL * (far ? root : 0.015625f), lower = far ? root : __uint_as_float((uint32_t)(127 + R) << 23);
        const float2 l2 = unpair(l[c >> 1]), v2 = unpair(vsum[c >> 1]);
        float lc = c & 1 ? l2.y : l2.x, vc = c & 1 ? v2.y : v2.x;
#pragma unroll
        for (int d = 4; d < 32; d *= 2) {
          lc += __shfl_xor_sync(0xffffffffu, lc, d);
          vc += __shfl_xor_sync(0xffffffffu, vc, d);
        }
#pragma unroll
        for (int w = 0; w < F::WV; w++)
#pragma unroll
          for (int j = 0; j < 4; j++) {
            float2 v;      // elements 2 j and 2 j + 1 of the word; the second stands 16 times too high
            v.x = fmaf(o[w][j][c >> 1][c & 1] * unit, lower, vc);
            v.y = fmaf(o[w][j][c >> 1][(c & 1) + 2] * (0.0625f * unit), lower, vc);
            *reinterpret_cast<float2*>(mine + r * (D + 4) + 8 * (F::WV * g + w) + 2 * j) = v;
          }
        if (g == 0) *reinterpret_cast<float2*>(mine + r * (D + 4) + D) = make_float2(reference(c), lc);
      }
    }
    __syncthreads();
    const bool complete = nt == s.tiles;
    const int bh = b * heads + h;
    float* slot = complete ? nullptr : fp.slots + (2ll * blockIdx.x + (t0 == 0 ? 1 : 0)) * F::SLOT;
    if (threadIdx.x == 0 && fp.split && t0 == 0) {
      // the last unit of this (sequence, head) lies with the block whose share holds it
      const int last = bh_unit + FLOW_SEGMENT + s.tiles - 1, even = longer * (share + 1);
      const int block = last < even ? last / (share + 1) : longer + (last - even) / share;
      fp.pieces[bh] = complete ? make_int2(0, 0) : make_int2((int)blockIdx.x, block - (int)blockIdx.x + 1);
    }
    for (int e = threadIdx.x; e < rows * (D / 4); e += 32 * FLOW_WARPS) {
      const int r = e / (D / 4), d = (e % (D / 4)) * 4;
      float M = -INFINITY;
      float2 ml[FLOW_WARPS];
#pragma unroll
      for (int w = 0; w < FLOW_WARPS; w++) {
        ml[w] = *reinterpret_cast<const float2*>(smem + w * F::PER_WARP + (r * (D + 4) + D) * 4);
        M = fmaxf(M, ml[w].x);
      }
      float L = 0.0f;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < FLOW_WARPS; w++) {
        // a warp that saw no key adds nothing; NaN scores keep l at NaN
        const float f = ml[w].x == -INFINITY ? (ml[w].y == 0.0f ? 0.0f : ml[w].y) : ex2(ml[w].x - M);
        if (ml[w].x == -INFINITY && ml[w].y == 0.0f) continue;
        const float4 x = *reinterpret_cast<const float4*>(smem + w * F::PER_WARP + (r * (D + 4) + d) * 4);
        L += f * ml[w].y;
        v.x += f * x.x;
        v.y += f * x.y;
        v.z += f * x.z;
        v.w += f * x.w;
      }
      if (complete) {
        finish_row<BF16, D>(p, s, h, r, d, M, L, v);
      } else {
        *reinterpret_cast<float4*>(slot + F::ROWS * 2 + r * D + d) = v;
        if (d == 0) *reinterpret_cast<float2*>(slot + r * 2) = make_float2(M, L);
      }
    }
    __syncthreads();     // the exchange area is the next segment's ring
    u = next_u;
    loc = 0;
    if (fp.split) h++;
  }
}

// Joins the partial results of the (sequence, head)s that lie in several blocks.  A warp takes one row and every WARPS-th piece
// of it, lanes over the row's elements; the warps meet in shared memory.  The order is fixed by the shares.
constexpr int JOIN_WARPS = 8;

template <bool BF16, int D, int NQ>
__global__ void __launch_bounds__(32 * JOIN_WARPS) kv4_attention_join_kernel(const FlowParams fp) {
  using F = Flow<D, NQ>;
  const AttentionParams& p = fp.a;
  constexpr int V = D / 128 > 0 ? D / 128 : 1;     // float4 per lane (D = 64: half the lanes)
  __shared__ float4 part_s[JOIN_WARPS][D / 4];
  __shared__ float2 ml_s[JOIN_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  const int bh = blockIdx.x, b = bh / p.cache.heads, h = bh - b * p.cache.heads;
  const int2 pc = __ldcg(fp.pieces + bh);      // on its way with the span's loads; what it holds without rows is not looked at
  const Span s = span_of<FLOW_TILE>(p, b);
  if (s.n <= 0 || pc.y == 0) return;
  for (int r = blockIdx.y; r < s.n * p.group; r += gridDim.y) {
    float M = -INFINITY, L = 0.0f;
    float4 v[V];
#pragma unroll
    for (int k = 0; k < V; k++) v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = warp; i < pc.y; i += JOIN_WARPS) {
      const float* slot = fp.slots + (2ll * (pc.x + i) + (i == 0 ? 1 : 0)) * F::SLOT;
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(slot + r * 2));
      float4 x[V];
#pragma unroll
      for (int k = 0; k < V; k++)
        if (D >= 128 || lane < D / 4) x[k] = __ldcg(reinterpret_cast<const float4*>(slot + F::ROWS * 2 + r * D) + k * 32 + lane);
      if (ml.x == -INFINITY && ml.y == 0.0f) continue;      // no key: nothing was written that counts
      const float top = fmaxf(M, ml.x);
      const float f = M == top ? 1.0f : ex2(M - top), g = ml.x == top ? 1.0f : ex2(ml.x - top);
      M = top;
      L = L * f + g * ml.y;
#pragma unroll
      for (int k = 0; k < V; k++)
        if (D >= 128 || lane < D / 4) {
          v[k].x = v[k].x * f + g * x[k].x;
          v[k].y = v[k].y * f + g * x[k].y;
          v[k].z = v[k].z * f + g * x[k].z;
          v[k].w = v[k].w * f + g * x[k].w;
        }
    }
#pragma unroll
    for (int k = 0; k < V; k++)
      if (D >= 128 || lane < D / 4) part_s[warp][k * 32 + lane] = v[k];
    if (lane == 0) ml_s[warp] = make_float2(M, L);
    __syncthreads();
    if (threadIdx.x < D / 4) {
      float top = -INFINITY, sum = 0.0f;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int w = 0; w < JOIN_WARPS; w++) top = fmaxf(top, ml_s[w].x);
      for (int w = 0; w < JOIN_WARPS; w++) {
        const float2 ml = ml_s[w];
        if (ml.x == -INFINITY && ml.y == 0.0f) continue;
        const float f = ml.x == top ? 1.0f : ex2(ml.x - top);
        const float4 x = part_s[w][threadIdx.x];
        sum += f * ml.y;
        o.x += f * x.x;
        o.y += f * x.y;
        o.z += f * x.z;
        o.w += f * x.w;
      }
      finish_row<BF16, D>(p, s, h, r, threadIdx.x * 4, top, sum, o);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------- host side
int largest_rows(int D) { return D == 256 ? 16 : 32; }    // of a sequence and key head on the flow kernel

struct FlowPlan {
  int nq, blocks, join, split;     // query rows / 8, grid, sequences * heads, whether a (sequence, head) may be split
  size_t pieces_at, slots_at, bytes;
};

FlowPlan flow_plan(const apnn_kv4_cache* c, const apnn_kv4_batch* b, int group) {
  FlowPlan f;
  const long long rows = (long long)b->max_q * group;
  f.nq = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
  const int D = c->head_dim;
  const int per_sm = f.nq == 1 ? (D == 256 ? Flow<256, 1>::BLOCKS : Flow<128, 1>::BLOCKS) : f.nq == 2 ? (D == 256 ? Flow<256, 2>::BLOCKS : Flow<128, 2>::BLOCKS) : Flow<128, 4>::BLOCKS;
  const long long keys = (long long)b->table_width * c->page_size;
  const long long whole = (long long)b->sequences * c->heads;
  f.split = keys > UNSPLIT_KEYS;
  const long long units = whole * ((keys + FLOW_TILE - 1) / FLOW_TILE + FLOW_SEGMENT);
  const long long most = (long long)device_sm_count() * per_sm;
  f.blocks = (int)(f.split ? (units < most ? units : most) : (whole < (1ll << 30) ? whole : 1ll << 30));
  f.join = (int)whole;
  f.pieces_at = 256;
  f.slots_at = (f.pieces_at + (f.split ? whole * 8 : 0) + 127) / 128 * 128;
  f.bytes = f.slots_at + (f.split ? 2ull * f.blocks * (8 * f.nq * (D + 2)) * 4 : 0);
  return f;
}

template <bool BF16, int D, int NQ>
apnn_status launch_flow(cudaStream_t stream, const FlowPlan& f, const FlowParams& fp) {
  const void* kernel = reinterpret_cast<const void*>(kv4_attention_flow_kernel<BF16, D, NQ>);
  cudaError_t e = ensure_max_smem(kernel, Flow<D, NQ>::SMEM);
  if (e != cudaSuccess) return cuda_fail(e, "kv4_attention_flow_kernel shared memory");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)f.blocks, 1, 1);
  cfg.blockDim = dim3(32 * FLOW_WARPS, 1, 1);
  cfg.dynamicSmemBytes = Flow<D, NQ>::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  cfg.numAttrs = pdl_attribute(attr);
  cfg.attrs = attr;
  e = cudaLaunchKernelEx(&cfg, kv4_attention_flow_kernel<BF16, D, NQ>, fp);
  if (e != cudaSuccess) return cuda_fail(e, "kv4_attention_flow_kernel");
  if (!f.split) return APNN_OK;
  int parts = 1;     // blocks that share the rows of a (sequence, head)
  while (parts < 8 * NQ && (long long)f.join * parts < 2 * device_sm_count()) parts *= 2;
  cfg.gridDim = dim3((unsigned)f.join, (unsigned)parts, 1);
  cfg.blockDim = dim3(32 * JOIN_WARPS, 1, 1);
  cfg.dynamicSmemBytes = 0;
  e = cudaLaunchKernelEx(&cfg, kv4_attention_join_kernel<BF16, D, NQ>, fp);
  return e == cudaSuccess ? APNN_OK : cuda_fail(e, "kv4_attention_join_kernel");
}

template <bool BF16, int D>
apnn_status launch_flow_rows(cudaStream_t stream, const FlowPlan& f, const FlowParams& fp) {
  if (f.nq == 1) return launch_flow<BF16, D, 1>(stream, f, fp);
  if (f.nq == 2) return launch_flow<BF16, D, 2>(stream, f, fp);
  if constexpr (D != 256) return launch_flow<BF16, D, 4>(stream, f, fp);
  return APNN_ERR_UNSUPPORTED;     // not reached: such rows take the other kernel
}

// What 32-bit positions and shares hold: tables of up to 2^30 positions, and tiles of all sequences and heads below 2^31.
constexpr int MOST_POSITIONS = 1 << 30;
bool too_long(const apnn_kv4_cache* c, const apnn_kv4_batch* b) {
  const long long keys = (long long)b->table_width * c->page_size;
  return keys > MOST_POSITIONS || (long long)b->sequences * c->heads * ((keys + FLOW_TILE - 1) / FLOW_TILE + FLOW_SEGMENT) > 0x7fffffffll;
}

}  // namespace
}  // namespace apnn

using namespace apnn;

extern "C" {

size_t apnn_kv4_attention_workspace_bytes(const apnn_kv4_cache* cache, const apnn_kv4_batch* batch, int q_heads) {
  Kv4View view = {};
  Kv4Batch geo = {};
  if (kv4_view(cache, &view) != APNN_OK || kv4_batch(batch, 1, &geo) != APNN_OK || q_heads <= 0 || q_heads % cache->heads != 0 ||
      q_heads > MOST_HEADS || too_long(cache, batch))
    return 0;
  const int group = q_heads / cache->heads;
  if ((long long)batch->max_q * group > largest_rows(cache->head_dim)) return kv4_prompt_workspace_bytes(cache, batch, group);
  return flow_plan(cache, batch, group).bytes;
}

apnn_status apnn_kv4_attention(void* stream, const apnn_kv4_cache* cache, const apnn_kv4_batch* batch,
                               const apnn_kv4_attention_args* a, void* workspace, size_t workspace_bytes) {
  AttentionParams p = {};
  if (!a || a->struct_size != sizeof(apnn_kv4_attention_args) || !a->q || !a->out) return APNN_ERR_INVALID_ARG;
  apnn_status st = kv4_view(cache, &p.cache);
  if (st == APNN_OK) st = kv4_batch(batch, a->rows, &p.batch);
  if (st != APNN_OK) return st;
  if (a->q_heads <= 0 || a->q_heads % cache->heads != 0) return APNN_ERR_INVALID_ARG;
  if (too_long(cache, batch) || a->q_heads > MOST_HEADS) return APNN_ERR_UNSUPPORTED;
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
  p.window = a->window < MOST_POSITIONS ? a->window : MOST_POSITIONS;      // as far as any row sees
  p.scale = a->scale;
  p.status_flag = static_cast<int*>(workspace);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if ((long long)batch->max_q * p.group <= largest_rows(cache->head_dim)) {
    const FlowPlan f = flow_plan(cache, batch, p.group);
    FlowParams fp = {p, reinterpret_cast<int2*>(static_cast<char*>(workspace) + f.pieces_at), reinterpret_cast<float*>(static_cast<char*>(workspace) + f.slots_at),
                     f.split, p.cache.page_shift < 5 ? p.cache.page_shift : 5};
    apnn_status (*const launch[2][3])(cudaStream_t, const FlowPlan&, const FlowParams&) = {
        {launch_flow_rows<false, 64>, launch_flow_rows<false, 128>, launch_flow_rows<false, 256>},
        {launch_flow_rows<true, 64>, launch_flow_rows<true, 128>, launch_flow_rows<true, 256>}};
    return launch[cache->type == APNN_TYPE_BF16][cache->head_dim / 128](s, f, fp);
  }
  return kv4_prompt(s, cache, batch, p, workspace);
}

apnn_status apnn_kv4_attention_check(void* stream, const void* workspace) {
  if (!workspace) return APNN_ERR_INVALID_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int flag = -1;
  cudaError_t e = cudaMemcpyAsync(&flag, workspace, sizeof(int), cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return cuda_fail(e, "apnn_kv4_attention_check");
  return flag == 0 ? APNN_OK : APNN_ERR_TIMEOUT;
}

}  // extern "C"
