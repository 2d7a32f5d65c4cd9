// Attention over the 4-bit cache for prompts: many rows of a sequence, on tcgen05.
//
// A block takes 256 rows (128 at D = 256) that share a key head -- the sequence's queries times the group -- against tiles of 128
// keys.  S = Q K^T and O += W V are tcgen05.mma kind::f16 with fp32 accumulators in TMEM; two row tiles of 128 take turns, so the
// tensor core works on one while the softmax of the other runs:
//   warps 0-3    spread: thread = key; levels to fp16 n - 8 (exact) in the swizzled operand tiles, K key by key (K-major), V as it lies
//                (its elements are the N dimension: MN-major).  A word's nibbles become pairs (0,4) (1,5) (2,6) (3,7) by masking; Q is
//                stored in the same order and the output put back in order at the end.
//   warps 4-11   softmax: thread = row; scores from TMEM, weights back into the columns the scores stood in (fp16, the A operand
//                of the second product), sums and the reference point in registers
//   warp 12      issues the MMAs, as a whole warp with uniform operands
// The scores' scale and offset belong to the key: s = scale (step_j (q . n_j) + low_j sum q), three packed operations for
// two scores, their parameters broadcast from shared memory.  Weights as on the flow kernel (kv4_attention.cu): they carry the value's step,
// relative to a reference point that follows the running maximum in steps of 2^8, so O is rescaled in TMEM only when it moves.  From
// the first tile on whose steps lie too far from those before, weights are taken against a second reference point of each row.
// Registers: 96 / 184 / 184 / 48 for the four warpgroups out of the 128 each was launched with (setmaxnreg; a thread keeps 128 scores).
// Bounds per 128 x 128 tile and 128 elements: 1024 clk of MMAs, 1024 of exponentials, about 950 issue slots of softmax and 200 of
// spreading (one K / V tile serves both row tiles).  Measured: 8192 tokens, 32 heads on 8, causal, 850 us, 647 TFLOP/s, 0.38 of the
// tensor cores' rate; a row tile's turn takes some 3100 clk, nearly all of it the one softmax warp a row tile has on a scheduler,
// whose loads, packed products, exponentials and roundings wait on one another (instructions issue in 44% of the cycles).  Sixteen
// softmax warps had too few registers for a row of scores and took 1.22 ms; scalar products in place of packed ones 1.02 ms.
// Few units and many keys: the keys are split over blocks and kv4_prompt_join_kernel adds the parts in order.
#include <type_traits>

#include "kv4_attention.cuh"

namespace apnn {
namespace {

using namespace tc5;

constexpr int TILE = 128;              // keys of a tile, rows of a row tile
constexpr int THREADS = 512;
constexpr int SLOTS = 4;               // tiles whose parameters are held
constexpr int MAX_SPLIT = 16;

template <int D>
struct Prompt {
  static constexpr int QT = D == 256 ? 1 : 2;             // row tiles of a block: O and S of each have to fit the 512 TMEM columns
  static constexpr int DEPTH = D == 256 ? 1 : 2;          // K tiles, and V tiles, in shared memory
  static constexpr int ROWS = TILE * QT;
  static constexpr int OPERAND = D / 64 * 16384;          // 128 rows of D fp16, in 64-element columns of 16 KiB
  static constexpr int K_AT = QT * OPERAND, V_AT = K_AT + DEPTH * OPERAND, PAR_AT = V_AT + DEPTH * OPERAND;
  // pairs of keys: (step, step, mid, mid) of the keys, of the values; then live bits (4 words), the largest steps (4), R, whether steps
  // lie far apart, and the smallest steps (4, at 48)
  static constexpr int SLOT = 2 * 64 * 16 + 64;
  static constexpr int BAR_AT = PAR_AT + SLOTS * SLOT;
  static constexpr int SMEM = BAR_AT + 256 + 1024;
  static constexpr int O_COLUMN = QT * TILE;              // S of the row tiles first
};

struct PromptParams {
  AttentionParams a;
  int blocks_q;          // blocks of rows of a sequence at most
  int split;
  float* parts;          // [unit][split][ROWS][D + 4] when split: o, then the reference point and the sum
};

__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t lead;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(lead));
  return lead;
}
// Four MMAs of 16 elements of K each; descriptors as low words, the high words are constants of the layouts.  A and B from shared
// memory (rows of 64 elements: 32 bytes further each time), or A from TMEM (8 columns further) and B sixteen keys further.
__device__ __forceinline__ void mma_ss4(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred q, p, t;\n\t.reg .b64 a, b;\n\t.reg .b32 al, bl;\n\t"
      "setp.ne.b32 q, %6, 0;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t"
      "add.u32 al, %1, 2;\n\tadd.u32 bl, %2, 2;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, t;\n\t"
      "add.u32 al, %1, 4;\n\tadd.u32 bl, %2, 4;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, t;\n\t"
      "add.u32 al, %1, 6;\n\tadd.u32 bl, %2, 6;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, t;\n\t}" ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void mma_ts4(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred q, p, t;\n\t.reg .b64 b;\n\t.reg .b32 al, bl;\n\t"
      "setp.ne.b32 q, %6, 0;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t"
      "add.u32 al, %1, 8;\n\tadd.u32 bl, %2, 128;\n\tmov.b64 b, {bl, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [al], b, %4, t;\n\t"
      "add.u32 al, %1, 16;\n\tadd.u32 bl, %2, 256;\n\tmov.b64 b, {bl, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [al], b, %4, t;\n\t"
      "add.u32 al, %1, 24;\n\tadd.u32 bl, %2, 384;\n\tmov.b64 b, {bl, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [al], b, %4, t;\n\t}" ::"r"(d), "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void commit_to(uint32_t bar, uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// (no memory clobber: loads of parameters may pass it; the wait below orders it)
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
      "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]));
}
__device__ __forceinline__ void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t at, uint32_t v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ uint32_t lds(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}
struct __align__(16) PairPair {      // of two keys: steps, mids
  Pair step, mid;
};
__device__ __forceinline__ uint32_t hadd2(uint32_t a, uint32_t b) {
  const __half2 v = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t mask_or(uint32_t a, uint32_t mask, uint32_t c) {      // (a & mask) | c in one instruction
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(mask), "r"(c));
  return d;
}
// Eight levels of a word -> pairs of n - 8: nibbles 0..3 and 4..7 side by side
__device__ __forceinline__ void spread8(uint32_t w, uint32_t (&o)[4]) {
  const uint32_t y = w >> 8;
  o[0] = hadd2(mask_or(w, 0x000f000fu, 0x64006400u), 0xe408e408u);      // 1024 + n - 1032
  o[1] = hadd2(mask_or(w, 0x00f000f0u, 0x54005400u), 0xd480d480u);      // 64 + n - 72
  o[2] = hadd2(mask_or(y, 0x000f000fu, 0x64006400u), 0xe408e408u);
  o[3] = hadd2(mask_or(y, 0x00f000f0u, 0x54005400u), 0xd480d480u);
}
// 2^e as a float, e within fp32's normal range
__device__ __forceinline__ float power2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// bits [lo, hi) of a word, clipped
__device__ __forceinline__ uint32_t bit_range(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  return hi <= lo ? 0u : (hi == 32 ? 0xffffffffu : (1u << hi) - 1u) & ~((1u << lo) - 1u);
}

template <bool BF16, int D>
__global__ void __launch_bounds__(THREADS, 1) kv4_prompt_kernel(const PromptParams pp) {
  using P = Prompt<D>;
  const AttentionParams& p = pp.a;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t bars = base + P::BAR_AT;
  const uint32_t q_full = bars;
  auto k_full = [&](int s) { return bars + 8u * (1 + s); };
  auto k_empty = [&](int s) { return bars + 8u * (3 + s); };
  auto v_full = [&](int s) { return bars + 8u * (5 + s); };
  auto v_empty = [&](int s) { return bars + 8u * (7 + s); };
  auto s_full = [&](int q) { return bars + 8u * (9 + q); };
  auto w_full = [&](int q) { return bars + 8u * (11 + q); };
  auto o_done = [&](int q) { return bars + 8u * (13 + q); };
  auto par_full = [&](int s) { return bars + 8u * (15 + s); };
  const uint32_t tmem_slot = bars + 8u * 20;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 4 * P::QT);
    for (int s = 0; s < 2; s++) {
      mbar_init(k_full(s), 4);
      mbar_init(k_empty(s), 1);
      mbar_init(v_full(s), 4);
      mbar_init(v_empty(s), 1);
      mbar_init(s_full(s), 1);
      mbar_init(w_full(s), 4);
      mbar_init(o_done(s), 1);
    }
    for (int s = 0; s < SLOTS; s++) mbar_init(par_full(s), 4);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = lds(tmem_slot);
  grid_dependency_wait();
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *p.status_flag = 0;

  // ---- this block's rows and keys: the last rows of the sequences first, they see the most keys
  const int part = (int)blockIdx.x % pp.split, bh = (int)blockIdx.x / pp.split;
  const int b = bh / p.cache.heads, h = bh - b * p.cache.heads;
  const int qb = pp.blocks_q - 1 - (int)blockIdx.y;
  const Span span = span_of<TILE>(p, b);
  const int all_rows = max(span.n, 0) * p.group, row0 = qb * P::ROWS;
  const int rows = min(all_rows - row0, P::ROWS);
  const bool any = rows > 0;
  const int tiles_q = rows > TILE ? 2 : 1;      // row tiles with rows
  int tile0 = 0, tiles = 0;
  int key_end = 0, key_begin = 0;
  if (any) {
    const int first = span.pos0 + row0 / p.group, last = span.pos0 + (row0 + rows - 1) / p.group;
    key_end = p.causal ? min(span.len, last + 1) : span.len;
    key_begin = p.causal && p.window > 0 ? max(0, first + 1 - p.window) : 0;
    tile0 = key_begin / TILE;
    const int all = key_end > key_begin ? (key_end + TILE - 1) / TILE - tile0 : 0;
    tile0 += (int)((long long)all * part / pp.split);
    tiles = (int)((long long)all * (part + 1) / pp.split) - (int)((long long)all * part / pp.split);
  }
  auto give_up = [&](int code) { atomicExch(p.status_flag, code); };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    // ---------------- spread ----------------
    const int key = threadIdx.x;      // of a tile
    const int* trow = p.batch.table + (long long)b * p.batch.table_stride;
    const int page_size = p.cache.page_size;
    const uint8_t* head = p.cache.data + h * p.cache.head_bytes;
    constexpr int CHUNKS = D / 32;    // 16-byte pieces of a row of levels
    // A tile ahead: the row's levels and parameters, of the keys and of the values; two ahead: where it lies (an offset to its slot in
    // the page's key levels, -1 where there is no row)
    uint4 words[2][CHUNKS];
    uint32_t par[2] = {0u, 0u};
    auto locate = [&](int i) -> long long {
      const int j = (tile0 + i) * TILE + key;
      if (i >= tiles || j >= key_end) return -1;      // key_end <= table_width * page_size
      const int id = __ldg(trow + (j >> p.cache.page_shift));
      return (uint32_t)id < (uint32_t)p.cache.pages ? id * p.cache.page_stride : -1;
    };
    auto fetch = [&](int which, int i, long long at) {
      const int slot = ((tile0 + i) * TILE + key) & (page_size - 1);
      const uint8_t* src = head + max(at, 0ll) + (long long)page_size * (D / 2) * which + (long long)slot * (D / 2);
#pragma unroll
      for (int c = 0; c < CHUNKS; c++)
        words[which][c] = at >= 0 ? __ldg(reinterpret_cast<const uint4*>(src) + c) : make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
      par[which] = at >= 0 ? __ldg(reinterpret_cast<const uint32_t*>(head + at + (long long)page_size * D + (which * page_size + slot) * 4ll)) : 0u;
    };
    auto store = [&](int which, uint32_t dst) {
      const uint32_t row = dst + (uint32_t)key * 128u, x = (uint32_t)(key & 7);
#pragma unroll
      for (int c = 0; c < CHUNKS; c++) {
        const uint32_t w[4] = {words[which][c].x, words[which][c].y, words[which][c].z, words[which][c].w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          uint32_t o[4];
          spread8(w[i], o);
          sts128(row + (uint32_t)(c >> 1) * 16384u + ((((uint32_t)(c & 1) * 4u + i) ^ x) << 4), o[0], o[1], o[2], o[3]);
        }
      }
    };
    bool ok = true;
    int R = -112;
    uint32_t under = 0xffffffffu;      // as steps_far_apart takes it
    long long at = locate(0), at1 = locate(1);
    fetch(0, 0, at);
    fetch(1, 0, at);
    // After a wait that ran out a warp announces nothing any more, but keeps meeting the other three at the barrier below, so that
    // all of them reach the end.
    for (int j = 0; j < tiles; j++) {
      const int s = j % P::DEPTH;
      const uint32_t ph = (uint32_t)(j / P::DEPTH) & 1u;
      const uint32_t slot_at = base + P::PAR_AT + (uint32_t)(j % SLOTS) * P::SLOT + (uint32_t)(key >> 1) * 16u + (uint32_t)(key & 1) * 4u;
      const long long at2 = locate(j + 2);
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(k_empty(s), ph ^ 1u));
      if (ok) {
        store(0, base + P::K_AT + s * P::OPERAND);
        const float2 f = unpack2<BF16>(par[0]);
        sts32(slot_at, __float_as_uint(f.x));
        sts32(slot_at + 8, __float_as_uint(fmaf(8.0f, f.x, f.y)));      // the value of level 8
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(k_full(s));
      }
      fetch(0, j + 1, at1);
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(v_empty(s), ph ^ 1u));
      const float2 f = unpack2<BF16>(par[1]);
      const uint32_t head_at = base + P::PAR_AT + (uint32_t)(j % SLOTS) * P::SLOT + 2048u;
      if (ok) {
        store(1, base + P::V_AT + s * P::OPERAND);
        const bool live = at >= 0;
        sts32(slot_at + 1024 + 8, __float_as_uint(fmaf(8.0f, f.x, f.y)));
        const uint32_t bits = __float_as_uint(fabsf(f.x));
        const uint32_t lives = __ballot_sync(0xffffffffu, live);
        const uint32_t counted = live && bits < 0x7f800000u && (tile0 + j) * TILE + key >= key_begin ? bits : 0u;
        const uint32_t most = __reduce_max_sync(0xffffffffu, counted), least = __reduce_min_sync(0xffffffffu, counted - 1u);
        if (lane == 0) {
          sts32(head_at + warp * 4, lives);
          sts32(head_at + 16 + warp * 4, most);
          sts32(head_at + 48 + warp * 4, least);
        }
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (ok) {
        // 2^R is above every value step met so far, within fp32's range: the largest of the four warps' keys
        const uint32_t all = max(max(lds(head_at + 16), lds(head_at + 20)), max(lds(head_at + 24), lds(head_at + 28)));
        R = max(R, min((int)(all >> 23) - 126, 127));
        under = min(under, min(min(lds(head_at + 48), lds(head_at + 52)), min(lds(head_at + 56), lds(head_at + 60))));
        const bool far = steps_far_apart(R, under);
        if (far) under = 0u;      // and from here on: R is -112 at least
        if (key == 0) {
          sts32(head_at + 32, (uint32_t)R);
          sts32(head_at + 36, far ? 1u : 0u);
        }
        uint32_t held = __float_as_uint(f.x * power2(6 - R));
        if (far) held = (__float_as_uint(__log2f(fabsf(f.x))) & ~1u) | (f.x < 0.0f ? 1u : 0u);      // log2, the sign in its lowest bit (2^-23 of an exponent)
        sts32(slot_at + 1024, held);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(v_full(s));
          mbar_arrive(par_full(j % SLOTS));
        }
      }
      fetch(1, j + 1, at1);
      at = at1;
      at1 = at2;
    }
    if (!ok && lane == 0) give_up(1);
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    // ---------------- softmax ----------------
    const int qt = (warp - 4) >> 2, r = ((warp & 3) << 5) | lane;
    if (qt < P::QT && any) {
      const int row = row0 + qt * TILE + r;                       // among the sequence's rows for this key head
      const bool live_row = row < all_rows;
      const int i = min(row, all_rows - 1) / p.group, g = row - i * p.group;      // g is used of live rows only
      const int pos = span.pos0 + i;
      const int end = p.causal ? min(span.len, pos + 1) : span.len;
      const int begin = p.causal && p.window > 0 ? pos + 1 - p.window : 0;
      const long long t = span.first + i;
      float qf, ql;
      {
        // the row as fp16 times a power of two (exact but for elements 2^28 below the largest), in the order of the levels
        const uint16_t* src = p.q + t * p.q_stride + (long long)(h * p.group + (live_row ? g : 0)) * D;
        float top = 0.0f, sum = 0.0f;
#pragma unroll 4
        for (int d = 0; d < D; d += 8) {
          const uint4 v = live_row ? __ldg(reinterpret_cast<const uint4*>(src + d)) : make_uint4(0u, 0u, 0u, 0u);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const float2 f = unpack2<BF16>(w[k]);
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
            sum += f.x + f.y;
          }
        }
        const int e = (int)(__float_as_uint(top) >> 23) - 127;
        const int shift = top > 0.0f && e < 128 ? 14 - max(e, -100) : 0;
        const float up = power2(shift);
        const uint32_t dst = base + (uint32_t)qt * P::OPERAND + (uint32_t)r * 128u, x = (uint32_t)(r & 7);
#pragma unroll 4
        for (int d = 0; d < D; d += 8) {
          const uint4 v = live_row ? __ldg(reinterpret_cast<const uint4*>(src + d)) : make_uint4(0u, 0u, 0u, 0u);
          const float2 a = unpack2<BF16>(v.x), c = unpack2<BF16>(v.y), u = unpack2<BF16>(v.z), w = unpack2<BF16>(v.w);
          sts128(dst + (uint32_t)(d >> 6) * 16384u + ((((uint32_t)d >> 3) & 7u) ^ x) * 16u, pack2<false>(a.x * up, u.x * up), pack2<false>(a.y * up, u.y * up),
                 pack2<false>(c.x * up, w.x * up), pack2<false>(c.y * up, w.y * up));
        }
        qf = p.scale * LOG2E * power2(-shift);
        ql = p.scale * LOG2E * sum;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);

      if (qt < tiles_q) {
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;          // this warp's quarter of the TMEM lanes
        const uint32_t s_at = tmem + lanes + (uint32_t)qt * TILE, o_at = tmem + lanes + P::O_COLUMN + (uint32_t)qt * D;
        const Pair qf2 = pair(qf, qf), ql2 = pair(ql, ql);
        Pair l[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)}, vsum[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)};      // two chains each
        float below = 0.0f, rise_at = -INFINITY;                    // minus the reference point (0: none yet), and 8 above it
        int R = -112;      // the values' steps come times 2^(6 - R)
        bool ok = true;
        int j = 0;
        auto rescale = [&](float k) {      // O of the row, behind the product that added to it last
          ok = __all_sync(0xffffffffu, mbar_wait(o_done(qt), (uint32_t)(j - 1) & 1u));
          if (!ok) return;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(o_at + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * k);
            tmem_st32(o_at + c, o);
          }
        };
        for (; j < tiles && ok; j++) {
          const uint32_t slot = base + P::PAR_AT + (uint32_t)(j % SLOTS) * P::SLOT;
          const PairPair* pars = reinterpret_cast<const PairPair*>(smem_raw + (slot - raw));      // keys, then values
          const int key = (tile0 + j) * TILE;
          ok = __all_sync(0xffffffffu, mbar_wait(par_full(j % SLOTS), (uint32_t)(j / SLOTS) & 1u) && mbar_wait(s_full(qt), (uint32_t)j & 1u));
          if (!ok || lds(slot + 2084) != 0u) break;
          tc_fence_after();
          float sc[TILE];
          tmem_ld32(s_at, *reinterpret_cast<uint32_t(*)[32]>(&sc[0]));
          uint32_t seen[4];
#pragma unroll
          for (int c = 0; c < 4; c++) seen[c] = lds(slot + 2048 + 4 * c) & bit_range(begin - key - 32 * c, end - key - 32 * c);
          const int rise = (int)lds(slot + 2080);
          const bool whole = __all_sync(0xffffffffu, (seen[0] & seen[1] & seen[2] & seen[3]) == 0xffffffffu);
          float top;
#pragma unroll
          for (int c = 0; c < 4; c++) {      // the next 32 columns are on their way while these are scaled
            tmem_ld_wait();
            if (c < 3) tmem_ld32(s_at + 32 * (c + 1), *reinterpret_cast<uint32_t(*)[32]>(&sc[32 * (c + 1)]));
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const int k = 32 * c + e;
              const Pair step = pars[k / 2].step, mid = pars[k / 2].mid;
              const float2 v = unpair(fma2(mul2(pair(sc[k], sc[k + 1]), step), qf2, mul2(mid, ql2)));
              sc[k] = v.x;
              sc[k + 1] = v.y;
            }
          }
          if (!whole) {
#pragma unroll
            for (int c = 0; c < TILE; c++)
              sc[c] = (seen[c >> 5] >> (c & 31)) & 1u ? sc[c] : -INFINITY;
          }
          {
            float most[8];
#pragma unroll
            for (int c = 0; c < 8; c++) most[c] = fmaxf(sc[c], sc[c + 8]);
#pragma unroll
            for (int c = 16; c < TILE; c += 8)
#pragma unroll
              for (int e = 0; e < 8; e++) most[e] = fmaxf(most[e], sc[c + e]);
            top = fmaxf(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])), fmaxf(fmaxf(most[4], most[5]), fmaxf(most[6], most[7])));
          }
          if (__any_sync(0xffffffffu, top > rise_at || rise != R)) {
            const float m = rise_at == -INFINITY ? -INFINITY : -below;
            const float shrink = power2(max(R - rise, -127));      // 2^-127 as 0
            R = rise;
            top = fmaxf(top, m);
            const float keep = m == top ? 1.0f : ex2(m - top);
            below = top == -INFINITY ? 0.0f : -top;
            rise_at = top + 8.0f;
#pragma unroll
            for (int c = 0; c < 2; c++) {
              l[c] = mul2(l[c], pair(keep, keep));
              vsum[c] = mul2(vsum[c], pair(keep, keep));
            }
            if (j > 0) {
              rescale(keep * shrink);
              if (!ok) break;
            }
          }
          const Pair below2 = pair(below, below);
          auto weigh = [&](auto tag) {      // apart for tiles without a masked key: no branch stands between the elements
            constexpr bool WHOLE = decltype(tag)::value;
#pragma unroll
            for (int c = 0; c < 4; c++) {
              uint32_t w[16];
#pragma unroll
              for (int e = 0; e < 16; e++) {
                const int k = 32 * c + 2 * e;
                const Pair step = pars[64 + k / 2].step, mid = pars[64 + k / 2].mid;
                const float2 z = unpair(add2(pair(sc[k], sc[k + 1]), below2));
                const Pair ex = pair(ex2(z.x), ex2(z.y));
                l[e & 1] = add2(l[e & 1], ex);
                float2 f = unpair(mul2(ex, step));
                if (WHOLE) {
                  vsum[e & 1] = fma2(ex, mid, vsum[e & 1]);
                } else {      // a masked place may hold NaN
                  const bool on0 = (seen[c] >> (2 * e)) & 1u, on1 = (seen[c] >> (2 * e + 1)) & 1u;
                  const float2 md = unpair(mid);
                  f.x = on0 ? f.x : 0.0f;
                  f.y = on1 ? f.y : 0.0f;
                  vsum[e & 1] = fma2(ex, pair(on0 ? md.x : 0.0f, on1 ? md.y : 0.0f), vsum[e & 1]);
                }
                w[e] = pack2<false>(f.x, f.y);
              }
              tmem_st16(s_at + 16 * c, w);      // columns of scores that were read
            }
          };
          if (whole) weigh(std::true_type());
          else weigh(std::false_type());
          tmem_st_done();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(w_full(qt));
        }
        // ---- the tiles from the first on whose steps lie far apart and come as their logarithms.  Two passes over the scores in TMEM, 32
        // columns at a time: weights of 32 columns take 16, which were read by then (4096 tokens, 32 heads on 8, D = 128: 390 us against
        // 240; with the scores in registers and the ordinary tiles' loop shared 434 and 280).
        const bool far = ok && j < tiles;
        float apart = far && rise_at != -INFINITY ? (float)(R - 6) : -INFINITY;      // the values' reference point less the softmax's
        for (; j < tiles && ok; j++) {
          const uint32_t slot = base + P::PAR_AT + (uint32_t)(j % SLOTS) * P::SLOT;
          const PairPair* pars = reinterpret_cast<const PairPair*>(smem_raw + (slot - raw));
          const int key = (tile0 + j) * TILE;
          ok = __all_sync(0xffffffffu, mbar_wait(par_full(j % SLOTS), (uint32_t)(j / SLOTS) & 1u) && mbar_wait(s_full(qt), (uint32_t)j & 1u));
          if (!ok) break;
          tc_fence_after();
          auto scores = [&](int c, float (&sc)[32]) -> uint32_t {      // of 32 keys, and which of them the row sees
            const uint32_t seen = lds(slot + 2048 + 4 * c) & bit_range(begin - key - 32 * c, end - key - 32 * c);
            __syncwarp();
            tmem_ld32(s_at + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&sc[0]));
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const Pair step = pars[16 * c + e / 2].step, mid = pars[16 * c + e / 2].mid;
              const float2 v = unpair(fma2(mul2(pair(sc[e], sc[e + 1]), step), qf2, mul2(mid, ql2)));
              sc[e] = (seen >> e) & 1u ? v.x : -INFINITY;
              sc[e + 1] = (seen >> (e + 1)) & 1u ? v.y : -INFINITY;
            }
            return seen;
          };
          float top = -INFINITY, most = -INFINITY;      // of the scores, and of them and the steps; NaN counts as none
#pragma unroll 1
          for (int c = 0; c < 4; c++) {
            float sc[32];
            scores(c, sc);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 z = unpair(add2(pair(sc[e], sc[e + 1]), pars[64 + 16 * c + e / 2].step));
              top = fmaxf(top, fmaxf(sc[e], sc[e + 1]));
              most = fmaxf(most, fmaxf(z.x, z.y));
            }
          }
          if (__any_sync(0xffffffffu, top > rise_at)) {
            const float m = rise_at == -INFINITY ? -INFINITY : -below;
            top = fmaxf(top, m);
            const float keep = m == top ? 1.0f : ex2(m - top);
            if (m != top) apart += m - top;      // the values' own point stays; -inf where no key was met
            below = top == -INFINITY ? 0.0f : -top;
            rise_at = top + 8.0f;
#pragma unroll
            for (int c = 0; c < 2; c++) {
              l[c] = mul2(l[c], pair(keep, keep));
              vsum[c] = mul2(vsum[c], pair(keep, keep));
            }
          }
          most += below;
          if (__any_sync(0xffffffffu, most > apart + 14.0f)) {
            const float up = fmaxf(apart, most - 6.0f), k = up == apart ? 1.0f : ex2(apart - up);
            apart = up;
            if (j > 0) {
              rescale(k);
              if (!ok) break;
            }
          }
          const float from = apart == -INFINITY ? 0.0f : -apart;
#pragma unroll 1
          for (int c = 0; c < 4; c++) {
            float sc[32];
            const uint32_t seen = scores(c, sc);
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const Pair step = pars[64 + 16 * c + e / 2].step;
              const float2 mid = unpair(pars[64 + 16 * c + e / 2].mid), lg = unpair(step);
              const Pair z = add2(pair(sc[e], sc[e + 1]), pair(below, below));
              const float2 z2 = unpair(z), x = unpair(add2(z, add2(step, pair(from, from))));
              const Pair ex = pair(ex2(z2.x), ex2(z2.y));
              const bool on0 = (seen >> e) & 1u, on1 = (seen >> (e + 1)) & 1u;      // a masked place may hold NaN
              l[0] = add2(l[0], ex);
              vsum[0] = fma2(ex, pair(on0 ? mid.x : 0.0f, on1 ? mid.y : 0.0f), vsum[0]);
              const float f0 = __uint_as_float(__float_as_uint(ex2(x.x)) | (__float_as_uint(lg.x) << 31));
              const float f1 = __uint_as_float(__float_as_uint(ex2(x.y)) | (__float_as_uint(lg.y) << 31));
              w[e / 2] = pack2<false>(on0 ? f0 : 0.0f, on1 ? f1 : 0.0f);
            }
            tmem_st16(s_at + 16 * c, w);
          }
          tmem_st_done();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(w_full(qt));
        }
        // ---- the row's output
        float total, mids;
        {
          const float2 a = unpair(add2(l[0], l[1])), c = unpair(add2(vsum[0], vsum[1]));
          total = a.x + a.y;
          mids = c.x + c.y;
        }
        if (tiles > 0 && ok) {
          ok = __all_sync(0xffffffffu, mbar_wait(o_done(qt), (uint32_t)(tiles - 1) & 1u));
          tc_fence_after();
        }
        if (!ok && lane == 0) give_up(2);
        if (ok) {
          const float m = rise_at == -INFINITY ? -INFINITY : -below;
          // the values' reference point in two factors: 2^(R - 6)
          const float root = ex2(0.5f * apart), unit = far ? root : power2(-6), lower = far ? root : power2(R);
          const bool none = total == 0.0f;      // no key seen
          const float inv = none ? 0.0f : 1.0f / total;
          float* part_row = pp.split > 1 ? pp.parts + ((((long long)bh * pp.blocks_q + qb) * pp.split + part) * P::ROWS + qt * TILE + r) * (D + 4) : nullptr;
          const int head = h * p.group + g;
          uint16_t* dst = p.out + t * p.out_stride + (long long)head * D;
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            __syncwarp();
            if (tiles > 0) {
              tmem_ld32(o_at + c, o);
              tmem_ld_wait();
            } else {
#pragma unroll
              for (int e = 0; e < 32; e++) o[e] = 0u;
            }
            if (!live_row) continue;
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              float f[8];
#pragma unroll
              for (int k = 0; k < 8; k++)      // element k of eight stands in column 2 (k % 4) + k / 4
                f[k] = none ? 0.0f : fmaf(__uint_as_float(o[e + 2 * (k & 3) + (k >> 2)]) * unit, lower, mids);
              if (pp.split > 1) {
                *reinterpret_cast<float4*>(part_row + c + e) = make_float4(f[0], f[1], f[2], f[3]);
                *reinterpret_cast<float4*>(part_row + c + e + 4) = make_float4(f[4], f[5], f[6], f[7]);
              } else {
                *reinterpret_cast<uint4*>(dst + c + e) = make_uint4(pack2<BF16>(f[0] * inv, f[1] * inv), pack2<BF16>(f[2] * inv, f[3] * inv),
                                                                    pack2<BF16>(f[4] * inv, f[5] * inv), pack2<BF16>(f[6] * inv, f[7] * inv));
              }
            }
          }
          if (live_row) {
            if (pp.split > 1) *reinterpret_cast<float2*>(part_row + D) = make_float2(m, total);
            else if (p.lse != nullptr) p.lse[t * p.q_heads + head] = none ? -INFINITY : m * LN2 + logf(total);
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    // ---------------- MMA ----------------
    if (warp == 12 && tiles > 0) {
      const uint32_t lead = elect_lane();
      constexpr uint32_t HI = (1024u >> 4) | (1u << 14) | (2u << 29);            // 8-row groups 1024 bytes apart, version, 128-byte swizzle
      constexpr uint32_t QK = (1u << 4) | ((uint32_t)(TILE >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24);                    // fp32 += fp16 x fp16
      constexpr uint32_t WV = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24);          // B is MN-major
      auto issue_qk = [&](int qt, int s) {
        const uint32_t a0 = ((base + qt * P::OPERAND) >> 4) | (1u << 16), b0 = ((base + P::K_AT + s * P::OPERAND) >> 4) | (1u << 16);
#pragma unroll
        for (int k = 0; k < D / 64; k++) mma_ss4(tmem + qt * TILE, a0 + k * (16384u >> 4), b0 + k * (16384u >> 4), HI, QK, k != 0 ? 1u : 0u, lead);
        commit_to(s_full(qt), lead);
      };
      bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0) && mbar_wait(k_full(0), 0));
      if (ok) {
        tc_fence_after();
        for (int qt = 0; qt < tiles_q; qt++) issue_qk(qt, 0);
        commit_to(k_empty(0), lead);
      }
      for (int j = 0; j < tiles && ok; j++) {
        const int s = j % P::DEPTH, n = (j + 1) % P::DEPTH;
        for (int qt = 0; qt < tiles_q && ok; qt++) {
          ok = __all_sync(0xffffffffu, mbar_wait(v_full(s), (uint32_t)(j / P::DEPTH) & 1u) && mbar_wait(w_full(qt), (uint32_t)j & 1u));
          if (!ok) break;
          tc_fence_after();
          // V: columns of 64 elements 16 KiB apart (the leading offset), eight keys 1024 bytes
          const uint32_t b0 = ((base + P::V_AT + s * P::OPERAND) >> 4) | ((16384u >> 4) << 16);
#pragma unroll
          for (int k = 0; k < TILE / 64; k++)
            mma_ts4(tmem + P::O_COLUMN + qt * D, tmem + qt * TILE + 32 * k, b0 + k * (8192u >> 4), HI, WV, (j | k) != 0 ? 1u : 0u, lead);
          commit_to(o_done(qt), lead);
          if (qt == tiles_q - 1) commit_to(v_empty(s), lead);
          if (j + 1 < tiles) {
            ok = __all_sync(0xffffffffu, mbar_wait(k_full(n), (uint32_t)((j + 1) / P::DEPTH) & 1u));
            if (!ok) break;
            tc_fence_after();
            issue_qk(qt, n);      // behind the product that reads the weights out of the same columns
            if (qt == tiles_q - 1) commit_to(k_empty(n), lead);
          }
        }
      }
      if (!ok && lane == 0) give_up(3);
    }
  }
  // ---------------- tear-down ----------------
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  grid_launch_dependents();
  if (warp == 12) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// Joins the parts of split rows, a warp a row.
template <bool BF16, int D>
__global__ void __launch_bounds__(256) kv4_prompt_join_kernel(const PromptParams pp) {
  using P = Prompt<D>;
  const AttentionParams& p = pp.a;
  const int lane = threadIdx.x & 31;
  grid_dependency_wait();
  const int bh = blockIdx.x, b = bh / p.cache.heads, h = bh - b * p.cache.heads;
  const Span span = span_of<TILE>(p, b);
  const int row = (int)blockIdx.y * 8 + (int)(threadIdx.x >> 5);
  if (row >= max(span.n, 0) * p.group) return;
  const float* src = pp.parts + (((long long)bh * pp.blocks_q + row / P::ROWS) * pp.split * P::ROWS + row % P::ROWS) * (D + 4);
  constexpr int V = D >= 128 ? D / 128 : 1;
  float M = -INFINITY, L = 0.0f;
  float4 v[V];
#pragma unroll
  for (int k = 0; k < V; k++) v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int i = 0; i < pp.split; i++) {
    const float* at = src + (long long)i * P::ROWS * (D + 4);
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(at + D));
    float4 x[V];
#pragma unroll
    for (int k = 0; k < V; k++)
      if (D >= 128 || lane < D / 4) x[k] = __ldcg(reinterpret_cast<const float4*>(at) + k * 32 + lane);
    if (ml.x == -INFINITY && ml.y == 0.0f) continue;
    const float top = fmaxf(M, ml.x);
    const float f = M == top ? 1.0f : ex2(M - top), g = ml.x == top ? 1.0f : ex2(ml.x - top);
    M = top;
    L = L * f + g * ml.y;
#pragma unroll
    for (int k = 0; k < V; k++)
      if (D >= 128 || lane < D / 4) v[k] = make_float4(v[k].x * f + g * x[k].x, v[k].y * f + g * x[k].y, v[k].z * f + g * x[k].z, v[k].w * f + g * x[k].w);
  }
#pragma unroll
  for (int k = 0; k < V; k++)
    if (D >= 128 || lane < D / 4) finish_row<BF16, D>(p, span, h, row, (k * 32 + lane) * 4, M, L, v[k]);
}

struct PromptPlan {
  int blocks_q, split;
  size_t bytes;
};

PromptPlan prompt_plan(const apnn_kv4_cache* c, const apnn_kv4_batch* b, int group) {
  PromptPlan f;
  const int D = c->head_dim, block_rows = D == 256 ? Prompt<256>::ROWS : Prompt<128>::ROWS;
  f.blocks_q = (int)(((long long)b->max_q * group + block_rows - 1) / block_rows);
  const long long units = (long long)b->sequences * c->heads * f.blocks_q;
  const long long tiles = ((long long)b->table_width * c->page_size + TILE - 1) / TILE;
  // enough parts for the device, four tiles to a part at least
  f.split = 1;
  while (f.split < MAX_SPLIT && units * f.split * 2 <= device_sm_count() && tiles >= 8 * f.split) f.split *= 2;
  f.bytes = 256 + (f.split > 1 ? (size_t)units * f.split * block_rows * (D + 4) * 4 : 0);
  return f;
}

template <bool BF16, int D>
apnn_status launch_prompt(cudaStream_t s, const PromptParams& p, int pairs) {
  const void* kernel = reinterpret_cast<const void*>(kv4_prompt_kernel<BF16, D>);
  cudaError_t e = ensure_max_smem(kernel, Prompt<D>::SMEM);
  if (e != cudaSuccess) return cuda_fail(e, "kv4_prompt_kernel shared memory");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(pairs * p.split), (unsigned)p.blocks_q, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = Prompt<D>::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  cfg.numAttrs = pdl_attribute(attr);
  cfg.attrs = attr;
  e = cudaLaunchKernelEx(&cfg, kv4_prompt_kernel<BF16, D>, p);
  if (e != cudaSuccess) return cuda_fail(e, "kv4_prompt_kernel");
  if (p.split == 1) return APNN_OK;
  cfg.gridDim = dim3((unsigned)pairs, (unsigned)(p.blocks_q * Prompt<D>::ROWS / 8), 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.dynamicSmemBytes = 0;
  e = cudaLaunchKernelEx(&cfg, kv4_prompt_join_kernel<BF16, D>, p);
  return e == cudaSuccess ? APNN_OK : cuda_fail(e, "kv4_prompt_join_kernel");
}

}  // namespace

size_t kv4_prompt_workspace_bytes(const apnn_kv4_cache* cache, const apnn_kv4_batch* batch, int group) { return prompt_plan(cache, batch, group).bytes; }

apnn_status kv4_prompt(cudaStream_t s, const apnn_kv4_cache* cache, const apnn_kv4_batch* batch, const AttentionParams& a, void* workspace) {
  const PromptPlan f = prompt_plan(cache, batch, a.group);
  if (f.blocks_q > 65535 || (long long)batch->sequences * cache->heads * f.split > 0x7fffffffll) return APNN_ERR_UNSUPPORTED;
  const PromptParams p = {a, f.blocks_q, f.split, reinterpret_cast<float*>(static_cast<char*>(workspace) + 256)};
  apnn_status (*const launch[2][3])(cudaStream_t, const PromptParams&, int) = {{launch_prompt<false, 64>, launch_prompt<false, 128>, launch_prompt<false, 256>},
                                                                               {launch_prompt<true, 64>, launch_prompt<true, 128>, launch_prompt<true, 256>}};
  return launch[cache->type == APNN_TYPE_BF16][cache->head_dim / 128](s, p, batch->sequences * cache->heads);
}

}  // namespace apnn
