// Matrix product over weight planes for more than a few rows of X, on tcgen05.
//
// The weights are the M operand of tcgen05.mma kind::f16 (128 of them to a block, 256 to a pair of blocks with cta_group::2), rows of X
// the N operand (tiles of 32 to 128, a pair's 256), so a thread of the epilogue owns one weight row: its scale and bias stay in registers and a warp
// stores 32 neighbouring columns of one row of the output.  X comes by TMA (128-byte swizzle, zeros beyond its edges), and so do the
// planes, 512 elements of K of every row at a time into a ring of two (loads of 8 bytes from 128 rows took as many L1
// cycles as a stage's MMAs: 0.74 against 0.43 ms at 4096 x 16384 x 4096, 4 bits).  The weights never exist as 16-bit floats in
// memory: groups of four warps spread the planes to level - zero (spread.cuh) and write the operand tile themselves, two stages of 64
// elements of K at a time, the groups in turn; a block alone keeps these tiles in TMEM, a pair swizzled in shared memory (its
// accumulators fill TMEM).  A warp that loads nothing meets each group on a named barrier and publishes the stages.  Roles: warp 0 TMA
// of X, 1 MMA, 2-9 epilogue (two to a quarter of the TMEM lanes), from 10 on spread, then publish and TMA of the planes; every wait
// is bounded.
//
// What bounds a stage: of the pair's 256 x 256 tile, shared memory, 32 KiB in and out for the weight tile and 256 bytes for each row
// of X a block holds, at 128 bytes a clock, 512 clk and as long as its MMAs (4096 x 16384 x 4096, 4 bits: 352 us, 1.56 PFLOP/s).  Of a
// block alone 0.15 us (1 bit) to 0.18 (4) whatever its width: the integer pipe, 240 clk at 4 bits, and the one warp that waits for
// stages, issues their MMAs and commits them (16 x 16384 x 4096, 2 bits: 13 us; with the tiles in shared memory 18.8).
//
// Few tiles and a long K: the blocks of a cluster share a tile's K, and each finishes a slice of the tile's rows of X from the others'
// sums in its shared memory, added in the order of the ranks.
#include <cstring>

#include "linear.cuh"

namespace apnn {
namespace {

using namespace tc5;

constexpr int ROWS = 128;                       // weight rows of a block
constexpr int MAX_STAGES = 8;
constexpr int A_BYTES = ROWS * BK;
constexpr int CHUNK = 8;                        // stages of 64 elements that one load of the planes covers
constexpr int PLANE_BYTES = ROWS * CHUNK * 8;   // of one plane
constexpr int CHUNKS = 2;
constexpr int EPI_WARPS = 8, FIRST_SPREAD = 2 + EPI_WARPS, GROUP_THREADS = 128;
// Groups of spreading warps.  A group that has spread a pair of stages waits for the slots of its next pair, 2 GROUPS stages on: with
// no fewer slots in the ring the use before the one it waits for is over by then, so the parity names one use only.  (128 x 4096 x 4096, 4
// bits, a block alone: 17.9 us with two groups, 16.7 with three, 16.0 with four; 1 bit 14.5, 14.0, 13.7.)
template <int CTAS>
struct Roles {
  static constexpr int GROUPS = CTAS == 2 ? 2 : 4, SPREAD_WARPS = 4 * GROUPS;
  static constexpr int PUBLISH = FIRST_SPREAD + SPREAD_WARPS, PLANES = PUBLISH + 1, THREADS = 32 * (PLANES + 1);
};
constexpr int COLUMNS = 16;                     // of an accumulator that an epilogue warp takes at a time
constexpr int SMEM_BYTES = 232448;              // all an SM has: alignment, barriers, planes, stages
constexpr int MAX_SPLIT = 8;
// TMEM columns between the two accumulators; a block alone keeps its weight tiles behind them, 32 columns for a stage
template <int CTAS>
constexpr int ACC_COLUMNS = CTAS == 2 ? 256 : 128;
constexpr int TILES_AT = 256, STAGE_COLUMNS = 32;
static_assert(TILES_AT + MAX_STAGES * STAGE_COLUMNS <= 512, "TMEM");

struct TileParams {
  LinearParams l;
  int tn;                   // rows of X in a tile (over the pair)
  int tiles_x, tiles_w;
  int kblocks;              // of 64 elements: even
  int split;                // blocks of a cluster that share K (1: none)
  int stages, stage_bytes;
  int wide;                 // 16-bit output whose pairs of columns are words
  uint32_t idesc;
};

__device__ __forceinline__ void arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// The same released to this block only: the publishing of a spread stage.  What it announces is read by the tensor core of the SM that
// wrote it, behind each writer's fence to the async proxy; no thread of the other block loads it, so nothing has to be made visible
// there (a release at cluster scope took 1000 clk a stage, twice the stage's MMAs).
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void named_arrive(int id, int count) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(count) : "memory"); }
__device__ __forceinline__ void named_sync(int id, int count) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(count) : "memory"); }
__device__ __forceinline__ void st_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// The four MMAs of a stage and the commit that frees it.  The whole warp runs this with uniform operands and one lane issues, so that
// descriptors stay in uniform registers: issued from a one-lane branch a stage took 600 clk whatever its width, more than the
// MMAs of a 256-wide tile.
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t lead;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(lead));
  return lead;
}
#define APNN_STAGE_MMAS(G)                                                                             \
  "{\n\t.reg .pred q, p, t;\n\t.reg .b64 a, b;\n\t.reg .b32 al, bl;\n\t"                                 \
  "setp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"                           \
  "mov.b64 a, {%1, %6};\n\tmov.b64 b, {%2, %6};\n\t"                                                     \
  "@q tcgen05.mma.cta_group::" G ".kind::f16 [%0], a, b, %3, p;\n\t"                                     \
  "add.u32 al, %1, 2;\n\tadd.u32 bl, %2, 2;\n\tmov.b64 a, {al, %6};\n\tmov.b64 b, {bl, %6};\n\t"         \
  "@q tcgen05.mma.cta_group::" G ".kind::f16 [%0], a, b, %3, t;\n\t"                                     \
  "add.u32 al, %1, 4;\n\tadd.u32 bl, %2, 4;\n\tmov.b64 a, {al, %6};\n\tmov.b64 b, {bl, %6};\n\t"         \
  "@q tcgen05.mma.cta_group::" G ".kind::f16 [%0], a, b, %3, t;\n\t"                                     \
  "add.u32 al, %1, 6;\n\tadd.u32 bl, %2, 6;\n\tmov.b64 a, {al, %6};\n\tmov.b64 b, {bl, %6};\n\t"         \
  "@q tcgen05.mma.cta_group::" G ".kind::f16 [%0], a, b, %3, t;\n\t}"
template <int CTAS>
__device__ __forceinline__ void stage_mmas(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
  constexpr uint32_t HI = (1024u >> 4) | (1u << 14) | (2u << 29);      // descriptor: 8-row groups 1024 bytes apart, version, 128-byte swizzle
  if (CTAS == 2) asm volatile(APNN_STAGE_MMAS("2") ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(lead), "r"(HI) : "memory");
  else asm volatile(APNN_STAGE_MMAS("1") ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(lead), "r"(HI) : "memory");
}
// The same with the weights in TMEM, 16 elements of K in 8 columns.
__device__ __forceinline__ void stage_mmas_tmem(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
  constexpr uint32_t HI = (1024u >> 4) | (1u << 14) | (2u << 29);
  asm volatile(
      "{\n\t.reg .pred q, p, t;\n\t.reg .b64 b;\n\t.reg .b32 al, bl;\n\t"
      "setp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "mov.b64 b, {%2, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t"
      "add.u32 al, %1, 8;\n\tadd.u32 bl, %2, 2;\n\tmov.b64 b, {bl, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [al], b, %3, t;\n\t"
      "add.u32 al, %1, 16;\n\tadd.u32 bl, %2, 4;\n\tmov.b64 b, {bl, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [al], b, %3, t;\n\t"
      "add.u32 al, %1, 24;\n\tadd.u32 bl, %2, 6;\n\tmov.b64 b, {bl, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [al], b, %3, t;\n\t}" ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(lead), "r"(HI)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
      "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
template <int CTAS>
__device__ __forceinline__ void commit(uint32_t bar, uint32_t lead) {      // pair: the barrier at this offset in both blocks
  if (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar), "h"((uint16_t)3), "r"(lead) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(lead) : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// One lane's copy of a box into shared memory, announced on `bar` (announce: with its bytes), by a whole warp with uniform operands
// for the same reason: from a one-lane branch a copy took 350 clk to issue, more than spreading a stage.
template <int CTAS>
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar, uint32_t lead) {
  if (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar), "r"(lead)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(dst), "l"(map), "r"(x),
        "r"(y), "r"(bar), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes, uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes), "r"(lead)
      : "memory");
}

// 16 columns of the epilogue: v[j] is the sum of weight row n (a lane each; live: there is one) with row m0 + j of X.  wide: the
// output may be stored in pairs of columns.
template <bool BF16>
__device__ __forceinline__ void finish_columns(const LinearParams& p, float (&v)[COLUMNS], long long m0, long long n, bool live, bool wide, float scale, float bias) {
  const int count = (int)min((long long)COLUMNS, (long long)p.M - m0);
  if (count <= 0) return;      // the whole warp
#pragma unroll
  for (int j = 0; j < COLUMNS; j++) v[j] = fmaf(v[j], scale, bias);
  switch (p.act) {
    case APNN_ACT_RELU:
#pragma unroll
      for (int j = 0; j < COLUMNS; j++) v[j] = activate(v[j], APNN_ACT_RELU);
      break;
    case APNN_ACT_SILU:
#pragma unroll
      for (int j = 0; j < COLUMNS; j++) v[j] = activate(v[j], APNN_ACT_SILU);
      break;
    case APNN_ACT_GELU:
#pragma unroll
      for (int j = 0; j < COLUMNS; j++) v[j] = activate(v[j], APNN_ACT_GELU);
      break;
    case APNN_ACT_GELU_TANH:
#pragma unroll
      for (int j = 0; j < COLUMNS; j++) v[j] = activate(v[j], APNN_ACT_GELU_TANH);
      break;
    default: break;
  }
  if (p.out_f32) {
    if (p.residual && live) {
      const float* r = static_cast<const float*>(p.residual) + m0 * p.ldr + n;
#pragma unroll
      for (int j = 0; j < COLUMNS; j++, r += p.ldr)
        if (j < count) v[j] += *r;
    }
    if (!live) return;
    float* o = static_cast<float*>(p.out) + m0 * p.ldo + n;
#pragma unroll
    for (int j = 0; j < COLUMNS; j++, o += p.ldo)
      if (j < count) *o = v[j];
    return;
  }
  if (p.residual && live) {
    const uint16_t* r = static_cast<const uint16_t*>(p.residual) + m0 * p.ldr + n;
    uint16_t x[COLUMNS];      // all on their way together: the stores below may be to the same addresses
#pragma unroll
    for (int j = 0; j < COLUMNS; j++, r += p.ldr) x[j] = j < count ? *r : (uint16_t)0;
#pragma unroll
    for (int j = 0; j < COLUMNS; j++) v[j] += unpack2<BF16>(x[j]).x;
  }
  uint16_t* o = static_cast<uint16_t*>(p.out) + m0 * p.ldo + n;
  if (wide) {
    // neighbouring lanes exchange a value of two rows, so that each stores two columns of one row
    const bool odd = threadIdx.x & 1;
    o += odd ? p.ldo - 1 : 0;
#pragma unroll
    for (int j = 0; j < COLUMNS; j += 2, o += 2 * p.ldo) {
      const float other = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[j + 1], 1);
      const uint32_t word = odd ? pack2<BF16>(other, v[j + 1]) : pack2<BF16>(v[j], other);
      if (live && j + (odd ? 1 : 0) < count) *reinterpret_cast<uint32_t*>(o) = word;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < COLUMNS; j++, o += p.ldo)
    if (live && j < count) *o = (uint16_t)pack2<BF16>(v[j], 0.0f);
}

// The named barrier on which a group hands over its pair of stages.  Two in turn for each group: it comes back to one only after the
// ring has let it reuse a slot, so after the publishing warp left it (4 GROUPS stages are more than a ring has).
template <int GROUPS>
__device__ __forceinline__ int group_barrier(uint32_t pair) { return 1 + (int)(pair % GROUPS * 2 + (pair / GROUPS & 1u)); }
static_assert(4 * Roles<1>::GROUPS >= MAX_STAGES && 4 * Roles<2>::GROUPS >= MAX_STAGES && 2 * Roles<1>::GROUPS < 16, "named barriers");

template <int WB, bool BF16, int CTAS>
__global__ void __launch_bounds__(Roles<CTAS>::THREADS, 1)
    linear_tile_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const TileParams p) {
  constexpr int STEP = CTAS == 2 ? 1 : 2;      // stages that share their barriers: the full one of the first, the empty one of the last
  constexpr int GROUPS = Roles<CTAS>::GROUPS, SPREAD_WARPS = Roles<CTAS>::SPREAD_WARPS, PUBLISH = Roles<CTAS>::PUBLISH, PLANES = Roles<CTAS>::PLANES;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t planes_at = base, stages_at = base + CHUNKS * WB * PLANE_BYTES, bars = stages_at + p.stages * p.stage_bytes;
  auto full_bar = [&](int s) { return bars + 8u * s; };                   // X landed and the weights are spread (in the leader)
  auto empty_bar = [&](int s) { return bars + 8u * (MAX_STAGES + s); };
  auto tfull_bar = [&](int a) { return bars + 8u * (2 * MAX_STAGES + a); };
  auto tempty_bar = [&](int a) { return bars + 8u * (2 * MAX_STAGES + 2 + a); };
  auto wfull_bar = [&](int c) { return bars + 8u * (2 * MAX_STAGES + 4 + c); };       // planes landed
  auto wempty_bar = [&](int c) { return bars + 8u * (2 * MAX_STAGES + 6 + c); };      // and were read by all spreading warps
  const uint32_t tmem_slot = bars + 8u * (2 * MAX_STAGES + 8);
  volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CTAS == 2 || p.split > 1 ? cluster_ctarank() : 0;
  const uint32_t half = CTAS == 2 ? rank : 0;                             // which rows of the pair's tile
  const int group = CTAS == 2 ? 2 : p.split;
  const int first_tile = blockIdx.x / group, tile_step = gridDim.x / group;
  const int num_tiles = p.tiles_x * p.tiles_w;
  // this block's blocks of K, an even number from an even one on
  const int kpairs = p.kblocks / 2;
  const int kb0 = CTAS == 1 ? 2 * (int)((long long)kpairs * rank / p.split) : 0;
  const int kbn = CTAS == 1 ? 2 * (int)((long long)kpairs * (rank + 1) / p.split) - kb0 : p.kblocks;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; s++) {
      mbar_init(full_bar(s), 1 + CTAS);   // the leader's TMA warp, the publishing warp of each block
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; a++) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), EPI_WARPS * CTAS);
      mbar_init(wfull_bar(a), 1);
      mbar_init(wempty_bar(a), SPREAD_WARPS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if (CTAS == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(512));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(512));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (CTAS == 2) cluster_sync_all();     // both blocks' barriers exist before anything remote touches them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot_ptr;
  grid_dependency_wait();
  if (p.l.status_flag && threadIdx.x == 0 && blockIdx.x == 0) *p.l.status_flag = 0;
  auto give_up = [&](int code) {
    if (p.l.status_flag) atomicExch(p.l.status_flag, code);
  };

  if (warp == 0) {
    // ---------------- X by TMA ----------------
    const uint32_t lead = elect_lane();
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    const int rows = p.tn / CTAS;
    for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
      const int row = tile % p.tiles_x * p.tn + (int)half * rows;
      for (int kb = 0; kb < kbn; kb += STEP) {
        if (!__all_sync(0xffffffffu, mbar_wait(empty_bar(s + STEP - 1), ph ^ 1u))) { ok = false; break; }
        if (CTAS == 1 || rank == 0) expect_bytes(full_bar(s), STEP * p.tn * BK, lead);     // pair of blocks: both blocks' bytes
#pragma unroll
        for (int i = 0; i < STEP; i++)
          copy_box<CTAS>(stages_at + (s + i) * p.stage_bytes + (CTAS == 2 ? A_BYTES : 0), &map_x, (kb0 + kb + i) * 64, row,
                         CTAS == 2 ? map_to_cta(full_bar(s), 0) : full_bar(s), lead);
        s = s + STEP == p.stages ? 0 : s + STEP;
        ph ^= s == 0 ? 1u : 0u;
      }
    }
    if (!ok && lane == 0) give_up(1);
  } else if (warp == 1) {
    // ---------------- MMA ----------------
    if (half == 0) {
      const uint32_t lead = elect_lane();
      int s = 0;
      uint32_t ph = 0, tl = 0;
      bool ok = true;
      for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step, tl++) {
        const uint32_t acc = tl & 1u;
        if (!__all_sync(0xffffffffu, mbar_wait(tempty_bar(acc), ((tl >> 1) & 1u) ^ 1u))) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * ACC_COLUMNS<CTAS>;
        for (int kb = 0; kb < kbn; kb += STEP) {
          if (!__all_sync(0xffffffffu, mbar_wait(full_bar(s), ph))) { ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < STEP; i++) {
            const uint32_t lo = ((stages_at + (s + i) * p.stage_bytes) >> 4) | (1u << 16);
            if (CTAS == 2) stage_mmas<CTAS>(d_tmem, lo, lo + (A_BYTES >> 4), p.idesc, kb + i != 0 ? 1u : 0u, lead);
            else stage_mmas_tmem(d_tmem, tmem_base + TILES_AT + (s + i) * STAGE_COLUMNS, lo, p.idesc, kb + i != 0 ? 1u : 0u, lead);
          }
          commit<CTAS>(empty_bar(s + STEP - 1), lead);
          s = s + STEP == p.stages ? 0 : s + STEP;
          ph ^= s == 0 ? 1u : 0u;
        }
        if (ok) commit<CTAS>(tfull_bar(acc), lead);
      }
      if (!ok && lane == 0) give_up(2);
    }
  } else if (warp == PLANES) {
    // ---------------- planes by TMA, a chunk ahead of the spreading ----------------
    const uint32_t lead = elect_lane();
    uint32_t chunk = 0;       // over all tiles
    bool ok = true;
    for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
      const int row = (tile / p.tiles_x * CTAS + (int)half) * ROWS;
      for (int kb = 0; kb < kbn; kb += CHUNK, chunk++) {
        const uint32_t c = chunk % CHUNKS;
        if (!__all_sync(0xffffffffu, mbar_wait(wempty_bar(c), ((chunk / CHUNKS) & 1u) ^ 1u))) { ok = false; break; }
        expect_bytes(wfull_bar(c), WB * PLANE_BYTES, lead);
        // rows behind N run into the next plane, and behind the last one they are zeros: their sums are not stored
#pragma unroll
        for (int b = 0; b < WB; b++)
          copy_box<1>(planes_at + (c * WB + b) * PLANE_BYTES, &map_w, 2 * (kb0 + kb), b * p.l.N + row, wfull_bar(c), lead);
      }
    }
    if (!ok && lane == 0) give_up(6);
  } else if (warp == PUBLISH) {
    // ---------------- publish spread stages ----------------
    const uint32_t full0 = CTAS == 2 ? map_to_cta(full_bar(0), 0) : map_to_cta(full_bar(0), rank);
    int s = 0;
    uint32_t pair = 0;        // of stages: the groups take them in turn
    for (int tile = first_tile; tile < num_tiles; tile += tile_step)
      for (int kb = 0; kb < kbn; kb += 2, pair++) {
        named_sync(group_barrier<GROUPS>(pair), GROUP_THREADS + 32);
#pragma unroll
        for (int i = 0; i < 2; i++, s = (s + 1 == p.stages) ? 0 : s + 1)
          if (lane == 0 && (i == 0 || STEP == 1)) arrive_remote(full0 + 8u * s);
      }
  } else if (warp >= FIRST_SPREAD) {
    // ---------------- spread the weights ----------------
    const uint32_t grp = (uint32_t)(warp - FIRST_SPREAD) >> 2;
    const int r = (warp & 3) * 32 + lane;      // a warp reaches a quarter of the TMEM lanes
    const ZeroPoint<BF16> zero(p.l.zero);
    const uint32_t row_at = stages_at + (uint32_t)r * 128u, xr = (uint32_t)(r & 7);
    const uint32_t words_at = planes_at + (uint32_t)r * 64u, wr = (uint32_t)(r >> 1) & 3u;      // 64-byte swizzle
    struct Slot { int s; uint32_t ph; } at = {0, 0};      // of the chunk's first stage
    auto after = [&](Slot x, int n) {
      for (x.s += n; x.s >= p.stages; x.s -= p.stages) x.ph ^= 1u;
      return x;
    };
    uint32_t pair = 0, chunk = 0;      // of the chunk's first pair
    bool ok = true;
    for (int tile = first_tile; tile < num_tiles; tile += tile_step) {
      for (int kc = 0; kc < kbn; kc += CHUNK, chunk++) {
        const uint32_t c = chunk % CHUNKS;
        const int count = min(CHUNK, kbn - kc) / 2;
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(wfull_bar(c), (chunk / CHUNKS) & 1u));
        // This group's pairs of the chunk.  (A loop over all pairs that skips the others' spread them all the same: the compiler
        // works ahead of the branch.)
        for (int i = (int)((grp + GROUPS - pair % GROUPS) % GROUPS); i < count; i += GROUPS) {
          uint4 words[WB];
#pragma unroll
          for (int b = 0; b < WB; b++) {
            const uint32_t from = words_at + (c * WB + b) * PLANE_BYTES + (((uint32_t)i ^ wr) << 4);
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(words[b].x), "=r"(words[b].y), "=r"(words[b].z), "=r"(words[b].w) : "r"(from));
          }
          const Slot one = after(at, 2 * i), two = after(one, 1);
          // the second stage's slot is freed after the first's.  After a wait that ran out the warp keeps meeting the named
          // barriers, so that everyone reaches the end
          if (ok) ok = __all_sync(0xffffffffu, mbar_wait(empty_bar(two.s), two.ph ^ 1u));
          if (ok) {
            if (CTAS == 1) tc_fence_after();
#pragma unroll
            for (int h = 0; h < 4; h++) {
              const int s = h < 2 ? one.s : two.s;
              uint32_t w[WB], o[16];
#pragma unroll
              for (int b = 0; b < WB; b++) w[b] = h == 0 ? words[b].x : h == 1 ? words[b].y : h == 2 ? words[b].z : words[b].w;
              spread_in_order<WB, BF16>(w, zero, o);
              if (CTAS == 1) {
                tmem_st16(tmem_base + ((uint32_t)(warp & 3) << 21) + TILES_AT + s * STAGE_COLUMNS + 16 * (h & 1), o);
              } else {
#pragma unroll
                for (int q = 0; q < 4; q++)
                  st_v4(row_at + s * p.stage_bytes + (((uint32_t)(4 * (h & 1) + q) ^ xr) << 4), o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
              }
            }
            if (CTAS == 1) {
              asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
              tc_fence_before();
            } else {
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            named_arrive(group_barrier<GROUPS>(pair + (uint32_t)i), GROUP_THREADS + 32);
          } else {
            named_sync(group_barrier<GROUPS>(pair + (uint32_t)i), GROUP_THREADS + 32);      // no ring holds it back: in step with the others
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(wempty_bar(c));
        at = after(at, 2 * count);
        pair += (uint32_t)count;
      }
    }
    if (!ok && lane == 0) give_up(4);
  } else if (CTAS == 2 || p.split == 1) {
    // ---------------- epilogue ----------------
    const int quarter = warp & 3, turn = (warp - 2) >> 2;
    uint32_t tl = 0;
    bool ok = true;
    for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step, tl++) {
      const uint32_t acc = tl & 1u;
      const long long n = ((long long)(tile / p.tiles_x) * CTAS + half) * ROWS + quarter * 32 + lane;
      const bool live = n < p.l.N;
      const bool wide = p.wide && n - lane + 32 <= p.l.N;      // all of the warp's columns
      const float scale = live ? __ldg(p.l.scale + n) : 0.0f, bias = live && p.l.bias ? __ldg(p.l.bias + n) : 0.0f;
      if (!__all_sync(0xffffffffu, mbar_wait(tfull_bar(acc), (tl >> 1) & 1u))) { ok = false; break; }
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * ACC_COLUMNS<CTAS>;
      const long long m0 = (long long)(tile % p.tiles_x) * p.tn;
#pragma unroll 1
      for (int c = turn * COLUMNS; c < p.tn; c += 2 * COLUMNS) {
        uint32_t v[COLUMNS];
        __syncwarp();
        tmem_ld16(taddr + c, v);
        tmem_ld_wait();
        float f[COLUMNS];
#pragma unroll
        for (int j = 0; j < COLUMNS; j++) f[j] = __uint_as_float(v[j]);
        finish_columns<BF16>(p.l, f, m0 + c, n, live, wide, scale, bias);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CTAS == 2) arrive_cluster(map_to_cta(tempty_bar(acc), 0));
        else mbar_arrive(tempty_bar(acc));
      }
    }
    if (!ok && lane == 0) give_up(3);
  }

  if (CTAS == 1 && p.split > 1) {
    // ---------------- the cluster's sums of one tile meet: every block's in the order of the ranks ----------------
    const bool reader = warp >= 2 && warp < 2 + EPI_WARPS;
    const int quarter = warp & 3, turn = (warp - 2) >> 2, slice = p.tn / p.split;      // rows of X that a rank finishes
    bool ok = true;
    __syncwarp();
    if (reader) ok = __all_sync(0xffffffffu, mbar_wait(tfull_bar(0), 0));
    if (!ok && lane == 0) give_up(5);
    tc_fence_after();
    cluster_sync_all();      // every block's MMAs have read their stages: the rings may be written over
    if (reader && ok) {
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
      for (int c = turn * COLUMNS; c < p.tn; c += 2 * COLUMNS) {
        uint32_t v[COLUMNS];
        __syncwarp();
        tmem_ld16(taddr + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < COLUMNS; j++) {
          const int col = c + j, owner = col / slice;
          // [rank that wrote][row of X within the slice][weight row]
          const uint32_t at = stages_at + (((uint32_t)rank * slice + (col - owner * slice)) * ROWS + quarter * 32 + lane) * 4u;
          asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(map_to_cta(at, owner)), "r"(v[j]) : "memory");
        }
      }
    }
    cluster_sync_all();
    if (reader && ok) {
      const int tile = first_tile;
      const long long n = (long long)(tile / p.tiles_x) * ROWS + quarter * 32 + lane;
      const bool live = n < p.l.N;
      const float scale = live ? __ldg(p.l.scale + n) : 0.0f, bias = live && p.l.bias ? __ldg(p.l.bias + n) : 0.0f;
      const long long m0 = (long long)(tile % p.tiles_x) * p.tn + (long long)rank * slice;
#pragma unroll 1
      for (int c = turn * 4; c < slice; c += 8) {
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          f[j] = 0.0f;
          for (int k = 0; k < p.split; k++)
            f[j] += *reinterpret_cast<const float*>(smem_raw + (stages_at - raw) + (((uint32_t)k * slice + c + j) * ROWS + quarter * 32 + lane) * 4u);
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (live && m0 + c + j < p.l.M) store_element<BF16>(p.l, m0 + c + j, n, f[j], scale, bias);
      }
    }
  }

  // ---------------- tear-down ----------------
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  grid_launch_dependents();
  if (CTAS == 2) cluster_sync_all();      // the peer may not leave while the leader's MMAs or arrivals can still reach it
  if (warp == 1) {
    tc_fence_after();
    if (CTAS == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512));
  }
}

// The plan of the shortest estimated time.  A wave of tiles takes its stages or its epilogue, whichever is longer, and the last
// epilogue shows; a split adds the exchange.  The figures (us) are fitted to 24 shapes on every plan (16 to 4096 rows, 1000 to 32003
// weights, K from 128 to 8192), most within a tenth: e.g. 333 x 2337 x 2296 13.2 on 64-wide tiles, 18.9 on the pair's 256;
// 32 x 4096 x 4096 10.9 with K in four, 18.0 without.
LinearPlan pick_plan(int M, int N, int kblocks, int sms) {
  LinearPlan best = {1, 32, 1};
  double least = 1e30;
  for (int ctas = 1; ctas <= 2; ctas++)
    for (int tn = ctas == 2 ? 256 : 32; tn <= 128 * ctas; tn *= 2)      // a pair: its full width alone, narrower ones were never shortest
      for (int split = 1; split <= (ctas == 2 ? 1 : MAX_SPLIT) && 2 * split <= kblocks; split *= 2) {
        if (tn / split < 4) continue;
        const long long tiles = (long long)((M + tn - 1) / tn) * ((N + ROWS * ctas - 1) / (ROWS * ctas));
        // a cluster finds its blocks within one group of SMs: the driver knows how many fit
        const int slots = split > 1 ? cluster_capacity(reinterpret_cast<const void*>(linear_tile_kernel<4, true, 1>), Roles<1>::THREADS, SMEM_BYTES, split) : sms / ctas;
        if (slots < 1) continue;
        const double stage = ctas == 1 ? (tn <= 64 ? 0.185 : 0.2) : 0.355;
        const double epilogue = (ctas == 1 ? 0.8 : 1.4) + 0.012 * tn;
        const double stages = stage * (double)((kblocks / 2 + split - 1) / split * 2);
        const double exchange = split > 1 ? 1.5 + 0.1 * (tn / split) + 0.015 * tn : 0.0;
        // a split block ends with its tile: the next wave's begins anew
        const double wave = split > 1 ? stages + exchange + epilogue + 3.0 : stages > epilogue ? stages : epilogue;
        const double time = (double)((tiles + slots - 1) / slots) * wave + (split > 1 ? 1.0 : 4.0 + epilogue);
        if (time < least) {
          least = time;
          best = {ctas, tn, split};
        }
      }
  return best;
}

template <int WB, bool BF16, int CTAS>
apnn_status launch(cudaStream_t s, const CUtensorMap& map, const CUtensorMap& map_w, const TileParams& p, int blocks) {
  const void* kernel = reinterpret_cast<const void*>(linear_tile_kernel<WB, BF16, CTAS>);
  cudaError_t e = ensure_max_smem(kernel, SMEM_BYTES);
  if (e != cudaSuccess) return cuda_fail(e, "linear_tile_kernel shared memory");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3(Roles<CTAS>::THREADS, 1, 1);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.numAttrs = pdl_attribute(attr);
  if (CTAS == 2 || p.split > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = CTAS == 2 ? 2u : (unsigned)p.split;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    cfg.numAttrs++;
  }
  cfg.attrs = attr;
  e = cudaLaunchKernelEx(&cfg, linear_tile_kernel<WB, BF16, CTAS>, map, map_w, p);
  return e == cudaSuccess ? APNN_OK : cuda_fail(e, "linear_tile_kernel");
}
template <bool BF16, int CTAS>
apnn_status launch_bits(cudaStream_t s, const CUtensorMap& map, const CUtensorMap& map_w, const TileParams& p, int blocks) {
  switch (p.l.wbits) {
    case 1: return launch<1, BF16, CTAS>(s, map, map_w, p, blocks);
    case 2: return launch<2, BF16, CTAS>(s, map, map_w, p, blocks);
    case 3: return launch<3, BF16, CTAS>(s, map, map_w, p, blocks);
    default: return launch<4, BF16, CTAS>(s, map, map_w, p, blocks);
  }
}

}  // namespace

LinearPlan linear_tile_plan(int M, int N, int kwords) { return pick_plan(M, N, kwords / 2, device_sm_count()); }

apnn_status linear_tile(cudaStream_t s, const LinearParams& l, bool bf16) {
  TileParams p = {};
  p.l = l;
  p.kblocks = l.kwords / 2;
  p.wide = !l.out_f32 && l.ldo % 2 == 0 && (reinterpret_cast<uintptr_t>(l.out) & 3u) == 0;
  const int sms = device_sm_count();
  const LinearPlan plan = linear_tile_plan(l.M, l.N, l.kwords);
  p.tn = plan.tn;
  p.split = plan.split;
  p.tiles_x = (l.M + plan.tn - 1) / plan.tn;
  p.tiles_w = (l.N + ROWS * plan.ctas - 1) / (ROWS * plan.ctas);
  // D = fp32, A and B = fp16 (0) or bf16 (1), K-major
  p.idesc = (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((uint32_t)(plan.tn >> 3) << 17) | ((uint32_t)(ROWS * plan.ctas >> 4) << 24);
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return cuda_fail(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
  CUtensorMap map;
  const cuuint64_t dims[2] = {(cuuint64_t)l.K, (cuuint64_t)l.M}, strides[1] = {(cuuint64_t)l.ldx * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)(plan.tn / plan.ctas)}, estr[2] = {1, 1};
  if (fn(&map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<uint16_t*>(l.X), dims, strides, box, estr,
         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cuda_fail(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
  CUtensorMap map_w;      // the planes one below the other, 64-byte rows of a chunk
  const cuuint64_t wdims[2] = {(cuuint64_t)l.kwords, (cuuint64_t)l.N * l.wbits}, wstrides[1] = {(cuuint64_t)l.kwords * 4};
  const cuuint32_t wbox[2] = {CHUNK * 2, ROWS};
  if (fn(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<uint32_t*>(l.W), wdims, wstrides, wbox, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cuda_fail(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
  p.stage_bytes = (plan.ctas == 2 ? A_BYTES : 0) + plan.tn / plan.ctas * BK;
  p.stages = (SMEM_BYTES - 2048 - CHUNKS * l.wbits * PLANE_BYTES) / p.stage_bytes;
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  if (plan.ctas == 1) p.stages &= ~1;
  if (p.stages < 2 * (plan.ctas == 2 ? Roles<2>::GROUPS : Roles<1>::GROUPS)) return APNN_ERR_UNSUPPORTED;      // not reached: 5 and 8 at least
  const long long tiles = (long long)p.tiles_x * p.tiles_w;
  const int slots = sms / plan.ctas;
  const int blocks = plan.split > 1 ? (int)tiles * plan.split : (int)(tiles < slots ? tiles : slots) * plan.ctas;
  if (plan.ctas == 2) return bf16 ? launch_bits<true, 2>(s, map, map_w, p, blocks) : launch_bits<false, 2>(s, map, map_w, p, blocks);
  return bf16 ? launch_bits<true, 1>(s, map, map_w, p, blocks) : launch_bits<false, 1>(s, map, map_w, p, blocks);
}

}  // namespace apnn
