// Matrix product over weight planes for more than a few rows of X, on tcgen05.
//
// The weights are the M operand of tcgen05.mma kind::f16 (128 of them to a block, 256 to a pair of blocks with cta_group::2), rows of X
// the N operand (tiles of 32 to 256), so a thread of the epilogue owns one weight row: its scale and bias stay in registers and a warp
// stores 32 neighbouring columns of one row of the output.  X comes by TMA (128-byte swizzle, zeros beyond its edges).  The
// weights never exist as 16-bit floats in memory: eight warps read the planes, spread them to level - zero (spread.cuh) and write
// the swizzled operand tile themselves, two groups of four warps on alternate stages of 64 elements of K; a warp that loads nothing
// meets each group on a named barrier and publishes the stage (a release at cluster scope waits for every load its warp has in
// flight).  Roles: warp 0 TMA, 1 MMA, 2-5 epilogue, 6-13 spread, 14 publish; every wait is bounded.
//
// What bounds a stage of 64 elements: shared memory, 32 KiB in and out for the weight tile and 256 bytes for each row of X a block
// holds, at 128 bytes a clock -- 512 clk for the pair's 256 x 256 tile, as long as its MMAs.  Spreading takes about 250.
//
// Few tiles and a long K: the blocks of a cluster share a tile's K, and each finishes a slice of the tile's rows of X from the others'
// sums in its shared memory, added in the order of the ranks.
#include <cstring>

#include "linear.cuh"

namespace apnn {
namespace {

using namespace tc5;

constexpr int ROWS = 128;                       // weight rows of a block
constexpr int STAGES = 6;
constexpr int A_BYTES = ROWS * BK, STAGE_BYTES = 2 * A_BYTES;
constexpr int SPREAD_WARPS = 8, GROUP_THREADS = 128;
constexpr int THREADS = 32 * (6 + SPREAD_WARPS + 1);
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 1024;
constexpr int MAX_SPLIT = 8;

struct TileParams {
  LinearParams l;
  int tn;                   // rows of X in a tile (over the pair)
  int tiles_x, tiles_w;
  int kblocks;              // of 64 elements: even
  int split;                // blocks of a cluster that share K (1: none)
  uint32_t idesc;
};

__device__ __forceinline__ void arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void named_arrive(int id, int count) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(count) : "memory"); }
__device__ __forceinline__ void named_sync(int id, int count) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(count) : "memory"); }
__device__ __forceinline__ void st_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity) {      // acquires what the peer's threads wrote
  unsigned long long t0 = 0;
  for (uint32_t spin = 0;; spin++) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    if ((spin & 255u) == 255u) {
      const unsigned long long now = global_timer_ns();
      if (t0 == 0) t0 = now;
      else if (now - t0 > WAIT_LIMIT_NS) return false;
    }
  }
}
template <int CTAS>
__device__ __forceinline__ void mma_f16_kind(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  if (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
template <int CTAS>
__device__ __forceinline__ void commit(uint32_t bar) {      // pair: the barrier at this offset in both blocks
  if (CTAS == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
  else
    tc_commit(bar);
}

// 32 columns of the epilogue: v[j] is the sum of weight row n with row m0 + j of X.
template <bool BF16>
__device__ __forceinline__ void finish_columns(const LinearParams& p, float (&v)[32], long long m0, long long n, bool live, float scale, float bias) {
  const int count = (int)min(32ll, (long long)p.M - m0);
  if (!live || count <= 0) return;
#pragma unroll
  for (int j = 0; j < 32; j++) v[j] = fmaf(v[j], scale, bias);
  switch (p.act) {
    case APNN_ACT_RELU:
#pragma unroll
      for (int j = 0; j < 32; j++) v[j] = activate(v[j], APNN_ACT_RELU);
      break;
    case APNN_ACT_SILU:
#pragma unroll
      for (int j = 0; j < 32; j++) v[j] = activate(v[j], APNN_ACT_SILU);
      break;
    case APNN_ACT_GELU:
#pragma unroll
      for (int j = 0; j < 32; j++) v[j] = activate(v[j], APNN_ACT_GELU);
      break;
    case APNN_ACT_GELU_TANH:
#pragma unroll
      for (int j = 0; j < 32; j++) v[j] = activate(v[j], APNN_ACT_GELU_TANH);
      break;
    default: break;
  }
  if (p.out_f32) {
    const float* r = static_cast<const float*>(p.residual) + m0 * p.ldr + n;
    float* o = static_cast<float*>(p.out) + m0 * p.ldo + n;
    if (p.residual) {
#pragma unroll
      for (int j = 0; j < 32; j++)
        if (j < count) v[j] += r[j * p.ldr];
    }
#pragma unroll
    for (int j = 0; j < 32; j++)
      if (j < count) o[j * p.ldo] = v[j];
  } else {
    const uint16_t* r = static_cast<const uint16_t*>(p.residual) + m0 * p.ldr + n;
    uint16_t* o = static_cast<uint16_t*>(p.out) + m0 * p.ldo + n;
    if (p.residual) {
#pragma unroll
      for (int j = 0; j < 32; j++)
        if (j < count) v[j] += unpack2<BF16>(r[j * p.ldr]).x;
    }
#pragma unroll
    for (int j = 0; j < 32; j++)
      if (j < count) o[j * p.ldo] = (uint16_t)pack2<BF16>(v[j], 0.0f);
  }
}

template <int WB, bool BF16, int CTAS>
__global__ void __launch_bounds__(THREADS, 1) linear_tile_kernel(const __grid_constant__ CUtensorMap map_x, const TileParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t bars = base + STAGES * STAGE_BYTES;
  auto full_bar = [&](int s) { return bars + 8u * s; };                   // X landed and the weights are spread (in the leader)
  auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
  auto tfull_bar = [&](int a) { return bars + 8u * (2 * STAGES + a); };
  auto tempty_bar = [&](int a) { return bars + 8u * (2 * STAGES + 2 + a); };
  const uint32_t tmem_slot = bars + 8u * (2 * STAGES + 4);
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
    for (int s = 0; s < STAGES; s++) {
      mbar_init(full_bar(s), 1 + CTAS);   // the leader's TMA warp, the publishing warp of each block
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; a++) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), 4 * CTAS);
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
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      const int rows = p.tn / CTAS;
      for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
        const int row = tile % p.tiles_x * p.tn + (int)half * rows;
        for (int kb = 0; kb < kbn; kb++, s = (s + 1 == STAGES) ? 0 : s + 1, ph ^= (s == 0) ? 1u : 0u) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u)) { ok = false; break; }
          const uint32_t dst = base + s * STAGE_BYTES + A_BYTES;
          if (CTAS == 2) {
            if (rank == 0) mbar_expect_tx(full_bar(s), p.tn * BK);     // both blocks' bytes
            tma_load_2d_pair(dst, &map_x, (kb0 + kb) * 64, row, map_to_cta(full_bar(s), 0));
          } else {
            mbar_expect_tx(full_bar(s), p.tn * BK);
            tma_load_2d(dst, &map_x, (kb0 + kb) * 64, row, full_bar(s));
          }
        }
      }
      if (!ok) give_up(1);
    }
  } else if (warp == 1) {
    // ---------------- MMA ----------------
    if (lane == 0 && half == 0) {
      int s = 0;
      uint32_t ph = 0, tl = 0;
      bool ok = true;
      for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step, tl++) {
        const uint32_t acc = tl & 1u;
        if (!mbar_wait(tempty_bar(acc), ((tl >> 1) & 1u) ^ 1u)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * 256;
        for (int kb = 0; kb < kbn; kb++, s = (s + 1 == STAGES) ? 0 : s + 1, ph ^= (s == 0) ? 1u : 0u) {
          if (!wait_cluster(full_bar(s), ph)) { ok = false; break; }
          tc_fence_after();
          const uint64_t adesc = make_smem_desc(base + s * STAGE_BYTES), bdesc = make_smem_desc(base + s * STAGE_BYTES + A_BYTES);
#pragma unroll
          for (int k = 0; k < 4; k++) mma_f16_kind<CTAS>(d_tmem, adesc + 2u * k, bdesc + 2u * k, p.idesc, (kb | k) != 0 ? 1u : 0u);
          commit<CTAS>(empty_bar(s));
        }
        if (ok) commit<CTAS>(tfull_bar(acc));
      }
      if (!ok) give_up(2);
    }
  } else if (warp == 6 + SPREAD_WARPS) {
    // ---------------- publish spread stages ----------------
    const uint32_t full0 = CTAS == 2 ? map_to_cta(full_bar(0), 0) : map_to_cta(full_bar(0), rank);
    int s = 0;
    uint32_t it = 0;
    for (int tile = first_tile; tile < num_tiles; tile += tile_step)
      for (int kb = 0; kb < kbn; kb++, it++, s = (s + 1 == STAGES) ? 0 : s + 1) {
        named_sync(1 + (int)((it & 1u) * 4 + ((it >> 1) & 3u)), GROUP_THREADS + 32);
        if (lane == 0) arrive_cluster(full0 + 8u * s);
      }
  } else if (warp >= 6) {
    // ---------------- spread the weights ----------------
    const int grp = (warp - 6) >> 2;
    const int r = ((warp - 6) & 3) * 32 + lane;
    const ZeroPoint<BF16> zero(p.l.zero);
    const uint32_t row_at = base + (uint32_t)r * 128u, xr = (uint32_t)(r & 7);
    int ftile = first_tile, fkb = grp;      // what is fetched next
    const uint32_t* src = nullptr;
    auto seek = [&]() {
      const long long n = ((long long)(ftile / p.tiles_x) * CTAS + half) * ROWS + r;
      src = p.l.W + min(n, (long long)p.l.N - 1) * p.l.kwords + 2 * kb0;      // rows behind N are not stored: they repeat the last
    };
    seek();
    auto fetch = [&](uint2 (&w)[WB]) {
      if (ftile >= num_tiles) return;
#pragma unroll
      for (int b = 0; b < WB; b++) w[b] = __ldg(reinterpret_cast<const uint2*>(src + b * p.l.plane_words + 2 * fkb));
      fkb += 2;
      if (fkb >= kbn) {
        fkb = grp;
        ftile += tile_step;
        if (ftile < num_tiles) seek();
      }
    };
    uint2 cur[WB] = {}, next[WB] = {};
    if (kbn > 0) fetch(cur);
    int s = grp;
    uint32_t ph = 0, it = 0;
    bool ok = true;
    for (int tile = first_tile; tile < num_tiles; tile += tile_step)
      for (int kb = grp; kb < kbn; kb += 2, it++) {
        fetch(next);
        // after a wait that ran out the warp keeps meeting the named barriers, so that everyone reaches the end
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(empty_bar(s), ph ^ 1u));
        if (ok) {
          const uint32_t dst = row_at + s * STAGE_BYTES;
#pragma unroll
          for (int h = 0; h < 2; h++) {
            uint32_t w[WB], o[16];
#pragma unroll
            for (int b = 0; b < WB; b++) w[b] = h ? cur[b].y : cur[b].x;
            spread_in_order<WB, BF16>(w, zero, o);
#pragma unroll
            for (int c = 0; c < 4; c++) st_v4(dst + (((uint32_t)(4 * h + c) ^ xr) << 4), o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        if (ok) named_arrive(1 + grp * 4 + (int)(it & 3u), GROUP_THREADS + 32);
        else named_sync(1 + grp * 4 + (int)(it & 3u), GROUP_THREADS + 32);      // no ring holds it back: in step with the others
#pragma unroll
        for (int b = 0; b < WB; b++) cur[b] = next[b];
        s += 2;
        if (s >= STAGES) {
          s -= STAGES;
          ph ^= 1u;
        }
      }
    if (!ok && lane == 0) give_up(4);
  } else if (CTAS == 2 || p.split == 1) {
    // ---------------- epilogue ----------------
    const int quarter = warp & 3;
    uint32_t tl = 0;
    bool ok = true;
    for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step, tl++) {
      const uint32_t acc = tl & 1u;
      const long long n = ((long long)(tile / p.tiles_x) * CTAS + half) * ROWS + quarter * 32 + lane;
      const bool live = n < p.l.N;
      const float scale = live ? __ldg(p.l.scale + n) : 0.0f, bias = live && p.l.bias ? __ldg(p.l.bias + n) : 0.0f;
      if (!__all_sync(0xffffffffu, mbar_wait(tfull_bar(acc), (tl >> 1) & 1u))) { ok = false; break; }
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * 256;
      const long long m0 = (long long)(tile % p.tiles_x) * p.tn;
#pragma unroll 1
      for (int c = 0; c < p.tn; c += 32) {
        uint32_t v[32];
        __syncwarp();
        tmem_ld32(taddr + c, v);
        tmem_ld_wait();
        float f[32];
#pragma unroll
        for (int j = 0; j < 32; j++) f[j] = __uint_as_float(v[j]);
        finish_columns<BF16>(p.l, f, m0 + c, n, live, scale, bias);
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
    const bool reader = warp >= 2 && warp < 6;
    const int quarter = warp & 3, slice = p.tn / p.split;      // rows of X that a rank finishes
    bool ok = true;
    __syncwarp();
    if (reader) ok = __all_sync(0xffffffffu, mbar_wait(tfull_bar(0), 0));
    if (!ok && lane == 0) give_up(5);
    tc_fence_after();
    cluster_sync_all();      // every block's MMAs have read their stages: the rings may be written over
    if (reader && ok) {
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < p.tn; c += 32) {
        uint32_t v[32];
        __syncwarp();
        tmem_ld32(taddr + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; j++) {
          const int col = c + j, owner = col / slice;
          // [rank that wrote][row of X within the slice][weight row]
          const uint32_t at = base + (((uint32_t)rank * slice + (col - owner * slice)) * ROWS + quarter * 32 + lane) * 4u;
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
      for (int c = 0; c < slice; c += 4) {
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          f[j] = 0.0f;
          for (int k = 0; k < p.split; k++)
            f[j] += *reinterpret_cast<const float*>(smem_raw + (base - raw) + (((uint32_t)k * slice + c + j) * ROWS + quarter * 32 + lane) * 4u);
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

struct Plan {
  int ctas, tn, split;
};

// The plan of the shortest estimated time, in clocks: waves of tiles times the stages of one, each as long as the slowest of the MMAs,
// shared memory and spreading, and what a block spends before its first stage and behind its last.
Plan pick_plan(int M, int N, int kblocks, int sms) {
  Plan best = {1, 32, 1};
  double least = 1e30;
  for (int ctas = 1; ctas <= 2; ctas++)
    for (int tn = ctas == 2 ? 64 : 32; tn <= 256; tn *= 2)
      for (int split = 1; split <= (ctas == 2 ? 1 : MAX_SPLIT) && 2 * split <= kblocks; split *= 2) {
        if (tn / split < 4) continue;
        const long long tiles = (long long)((M + tn - 1) / tn) * ((N + ROWS * ctas - 1) / (ROWS * ctas));
        const int slots = sms / (ctas * split);
        const double stage = 2.0 * tn > 256.0 + 2.0 * tn / ctas ? 2.0 * tn : 256.0 + 2.0 * tn / ctas;
        const double stages = (double)((kblocks / 2 + split - 1) / split * 2);
        const double time = (double)((tiles + slots - 1) / slots) * (stages * (stage > 300 ? stage : 300) + (split > 1 ? 3000.0 + 20.0 * tn : 0.0)) + 4000.0 + 15.0 * tn;
        if (time < least) {
          least = time;
          best = {ctas, tn, split};
        }
      }
  return best;
}

template <int WB, bool BF16, int CTAS>
apnn_status launch(cudaStream_t s, const CUtensorMap& map, const TileParams& p, int blocks) {
  const void* kernel = reinterpret_cast<const void*>(linear_tile_kernel<WB, BF16, CTAS>);
  cudaError_t e = ensure_max_smem(kernel, SMEM_BYTES);
  if (e != cudaSuccess) return cuda_fail(e, "linear_tile_kernel shared memory");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
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
  e = cudaLaunchKernelEx(&cfg, linear_tile_kernel<WB, BF16, CTAS>, map, p);
  return e == cudaSuccess ? APNN_OK : cuda_fail(e, "linear_tile_kernel");
}
template <bool BF16, int CTAS>
apnn_status launch_bits(cudaStream_t s, const CUtensorMap& map, const TileParams& p, int blocks) {
  switch (p.l.wbits) {
    case 1: return launch<1, BF16, CTAS>(s, map, p, blocks);
    case 2: return launch<2, BF16, CTAS>(s, map, p, blocks);
    case 3: return launch<3, BF16, CTAS>(s, map, p, blocks);
    default: return launch<4, BF16, CTAS>(s, map, p, blocks);
  }
}

}  // namespace

apnn_status linear_tile(cudaStream_t s, const LinearParams& l, bool bf16) {
  TileParams p = {};
  p.l = l;
  p.kblocks = l.kwords / 2;
  const int sms = device_sm_count();
  const Plan plan = pick_plan(l.M, l.N, p.kblocks, sms);
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
  const long long tiles = (long long)p.tiles_x * p.tiles_w;
  const int slots = sms / plan.ctas;
  const int blocks = plan.split > 1 ? (int)tiles * plan.split : (int)(tiles < slots ? tiles : slots) * plan.ctas;
  if (plan.ctas == 2) return bf16 ? launch_bits<true, 2>(s, map, p, blocks) : launch_bits<false, 2>(s, map, p, blocks);
  return bf16 ? launch_bits<true, 1>(s, map, p, blocks) : launch_bits<false, 1>(s, map, p, blocks);
}

}  // namespace apnn
