// Matrix products of block-scaled e4m3 operands: C[m, n] = epilogue(sum over blocks b of 128 along K of
// a_scale[b, m] * b_scale[n / 128, b] * (A[m, block b] . B[n, block b])), dense and grouped by expert.
//
// The scales are any f32 and change along the contraction, so the tensor cores sum one block only: four MMAs (32 of K each) fill one of four
// TMEM buffers of BN columns (one of two with 256), and while they fill the next ones, eight warps read it and add it, scaled, to sums in registers (f32; two
// warps share a TMEM lane quarter, a thread has half a row).  A block of K is one stage of the operand ring: 128 rows x 128 bytes of A,
// BN x 128 of B.  When the last block is in, the sums go back to TMEM, from where the plain epilogue takes them 16 columns at a time.
//
// What bounds the main loop is how fast the warps get through their instructions (clocks a block of K, 512 x 2048 x 8192):
//   - the MMA thread took 366 with divisions by the number of stages and waits asked for when they were due, whatever the width: its loop
//     counts up, asks for the next stage and buffer before it issues, and is unrolled, since an MMA holds its descriptors' registers until
//     the tensor core takes it (269 -> 150 - 190 without the sums);
//   - the warps that sum took 865 with the scales loaded four blocks ahead (a load waits behind the operands, over 1000 clocks), 580 - 690
//     with 16 warps of half the columns (what every warp does once a block filled the schedulers), and take 330 (64 columns) and 420 (128).
// 24.5 -> 16.4 us (64) and 28.3 -> 18.6 us (128) at that size.  With all SMs at work the operands' way out of L2 is a bound beside it: a block of 128 columns, 32 KB a
// CTA, takes 540 clocks then (13.4 TB/s).  256 columns, 840 clocks, need a quarter less of it and half the epilogues: they win where K is short, 128 where it is
// long.  8192 x 8192, us in 128 / 256 columns: K = 512 92 - 102 / 80, 1024 115 - 120 / 106 - 111, 2048 180 - 207 / 181 - 212, 4096 324 - 338 / 372 - 409,
// 8192 603 - 651 / 633 - 699 (1.7 - 1.9 PFLOP/s, at the clock that the power limit leaves); 4096^3 74 / 78 - 93.
//
// A CTA stays for all tiles of its share: while its warps are in the epilogue of one, the copies and the MMAs of the next go on (8192^3 814 -> 632 us,
// 512 x 8192 x 2048 narrowed with SiLU 21.9 -> 17.4 with that, tiles of 256 columns and results narrowed from registers).  A tile begins with buffer 0 and its epilogue
// keeps the last block's, so where that is buffer 0 too (4 i + 1 blocks; with 256 columns an odd number) the next tile's first products wait for the epilogue.
// Warp 0 TMA, warp 1 MMA, warps 2-9 (4-11 with 256 columns) sums and epilogue.  K slices are the CTAs of a cluster, as in gemm.cu (64-column tiles).
#include <atomic>

#include "gemm_common.cuh"

namespace qb {

constexpr int kSumWarps = 8;
constexpr int kSumThreads = 32 * kSumWarps;
constexpr int kColGroups = kSumWarps / 4;  // warps that share a TMEM lane quarter, each with its columns

// 256 columns: a thread has 128 sums beside what is on its way.  The control warps are a warpgroup of their own then, which hands
// registers over (setmaxnreg): an increase waits until that many are free, so the shares have to fit what the launch was given.
constexpr int kWideThreads = 384, kWideLaunchRegs = 168, kWideCtrlRegs = 56, kWideSumRegs = 224;
static_assert(128 * kWideCtrlRegs + kSumThreads * kWideSumRegs <= kWideThreads * kWideLaunchRegs, "register budget of the CTA");
template <int BN>
constexpr int kFirstSumWarp = BN == 256 ? 4 : 2;
template <int BN>
constexpr int kBlockThreads = 32 * kFirstSumWarp<BN> + kSumThreads;

struct BlockArgs {
  GemmArgs g;
  const float* a_scale;  // [kb_total][M]
  const float* b_scale;  // [N / 128 (of every expert)][kb_total]
  float* c_scale;        // [N / 128][M], e4m3 C
  const int* tile_rows;  // grouped: slots of a tile that hold a token
  int pow2, n_experts;
  int small_rows;  // rows of A in the box of the second map (grouped)
};

template <int BN>
struct BlockSmem {
  static constexpr int kStageBytes = (kBM + BN) * kRowBytes;  // a block of K: the rows of A, then those of B
  static constexpr int kSliceBytes = BN == 64 ? kBM * BN * 4 : 0;  // partial sums that the cluster's other K slices push
  static constexpr int kStages = BN == 64 ? 7 : BN == 128 ? 6 : 4;
  static constexpr int kAccBuffers = BN == 256 ? 2 : 4;  // of a block's products in TMEM
  static constexpr int kSliceOffset = kStages * kStageBytes;
  static constexpr int kBarOffset = kSliceOffset + kSliceBytes;
  static constexpr int kColOffset = kBarOffset + 256;  // per-column scale (unused), bias, gate
  static constexpr int kTopOffset = kColOffset + 3 * BN * 4;
  static constexpr int kTotal = kTopOffset + kColGroups * kBM * 4 + 1024;  // + alignment slack
  static_assert((2 * kStages + kAccBuffers + 1) * 8 + 32 <= 256 && kTotal <= 227 * 1024, "shared memory of one CTA");
};

__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld32(taddr, r); }
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld16(taddr, r); }

__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[32]) { tmem_st32(taddr, r); }
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[16]) { tmem_st16(taddr, r); }

// d += a * b on two f32 at once
__device__ __forceinline__ void fma2(float2& d, float ax, float ay, float2 b) {
  asm("{\n\t.reg .b64 p, q, r;\n\t"
      "mov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tmov.b64 r, {%4, %5};\n\t"
      "fma.rn.f32x2 p, q, r, p;\n\t"
      "mov.b64 {%0, %1}, p;\n\t}"
      : "+f"(d.x), "+f"(d.y)
      : "f"(ax), "f"(ay), "f"(b.x), "f"(b.y));
}

template <int BN, bool GROUPED>
__global__ void __launch_bounds__(kBlockThreads<BN>, 1)
gemm_blocks_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA_small, const __grid_constant__ CUtensorMap tmB, const BlockArgs args) {
  using L = BlockSmem<BN>;
  constexpr int kStages = L::kStages;
  constexpr int kAccBuffers = L::kAccBuffers, kW0 = kFirstSumWarp<BN>;
  constexpr int kScales = BN == 256 ? 4 : 8;  // blocks whose scales a thread has on their way
  constexpr uint32_t kTmemCols = kAccBuffers * BN;
  constexpr uint32_t kIdesc = umma_idesc(0, 0, kBM, BN);
  constexpr int kCols = BN / kColGroups;  // columns of a thread
  const GemmArgs& g = args.g;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::kBarOffset);
  // [stage] the MMAs that read the stage are done: it may be filled again, and their products are complete.  (The barrier cannot be a
  // phase ahead of a warp that sums: the stage's next MMAs come kStages blocks later, behind the sums of the block kAccBuffers before.)
  uint64_t* empty_bar = full_bar + kStages;
  static_assert(kStages >= kAccBuffers, "see above");
  uint64_t* acc_empty = empty_bar + kStages;      // [buffer] the warps that sum have read a block's products
  uint64_t* drain_bar = acc_empty + kAccBuffers;  // the MMAs in flight when the CTA gives up are done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* drain_flag = abort_flag + 1;  // never set: lets the drain waits below run their own limit
  volatile int* lost_flag = abort_flag + 2;   // set by a CTA of the cluster whose slice is missing
  float* col = reinterpret_cast<float*>(smem + L::kColOffset);
  float* tops = reinterpret_cast<float*>(smem + L::kTopOffset);  // 128 columns: [column group][row], largest magnitude of a thread's columns

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.z;
  const int kb0 = split * g.kb_per_split, n_iter = min(kb0 + g.kb_per_split, g.kb_total) - kb0;
  const bool clustered = BN == 64 && g.cluster != 0;  // one tile per cluster
  if (GROUPED) {
    grid_dep_wait();  // the tables are written by the routing kernel
    grid_dep_launch();
  }
  // Where tile t of the walk lies; false for one without tokens.  Dense: groups of 8 row tiles, the row index fastest, so that what runs at the
  // same time shares row tiles of A and column tiles of B.  Grouped: the columns of a row tile together.
  const int tiles_n = g.n_tiles / g.tiles_m;
  auto locate = [&](int t, int& m0, int& n0, int& rows, int& expert) {
    int mt, nt;
    if (GROUPED) {
      mt = t / tiles_n;
      nt = t - mt * tiles_n;
    } else {
      const int group = t / (8 * tiles_n), gm = min(g.tiles_m - 8 * group, 8), i = t - group * 8 * tiles_n;
      nt = i / gm;
      mt = 8 * group + i - nt * gm;
    }
    m0 = mt * kBM;
    n0 = nt * BN;
    expert = 0;
    rows = min(g.M - m0, kBM);
    if (GROUPED) {
      expert = after_wait(g.tile_expert)[mt];
      rows = min(after_wait(args.tile_rows)[mt], kBM);
      return expert >= 0 && expert < args.n_experts && rows > 0;
    }
    return true;
  };

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    for (int b = 0; b < kAccBuffers; ++b) mbar_init(smem_u32(&acc_empty[b]), kSumWarps);
    mbar_init(smem_u32(drain_bar), 1);
    *abort_flag = 0;
    *drain_flag = 0;
    *lost_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  if (clustered) cluster_sync();  // every CTA of the cluster is there before anyone pushes to it
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (!GROUPED) grid_dep_launch();

  if (BN == 256 && warp < kW0) setmaxnreg_dec<kWideCtrlRegs>();
  if (warp == 0) {
    // ---------------- TMA producer
    if (elect_one()) {
      const uint32_t full0 = smem_u32(full_bar), empty0 = smem_u32(empty_bar), stage0 = smem_u32(smem);
      int s = 0;
      uint32_t ph = 1;  // (a fresh barrier passes for parity 1)
      bool alive = true, waited = GROUPED;
      for (int t = blockIdx.x; t < g.n_tiles && alive; t += gridDim.x) {
        int m0, n0, rows, expert;
        if (!locate(t, m0, n0, rows, expert)) continue;
        const bool small = GROUPED && rows <= args.small_rows;
        const CUtensorMap* a_map = small ? &tmA_small : &tmA;
        const uint32_t stage_tx = (small ? args.small_rows : g.a_rows) * kRowBytes + BN * kRowBytes;
        const int b_row0 = expert * g.N + n0;
        int it = 0;
        if (!waited) {
          // constant weights do not depend on the kernels before this one: their first tiles are on the way while those finish
          // (four of them, since the first rows of A queue behind: one row of 8192 x 2048 7.5 -> 7.3 us, 512 x 2048 x 8192 16.3 -> 16.1 against all stages)
          const int ahead = g.b_const ? min(4, n_iter) : 0;
          for (; it < ahead; ++it) {
            mbar_arrive_expect_tx(full0 + it * 8, stage_tx);
            tma_load_2d(stage0 + it * L::kStageBytes + kBM * kRowBytes, &tmB, full0 + it * 8, (kb0 + it) * 128, b_row0);
          }
          grid_dep_wait();
          for (int i = 0; i < ahead; ++i) tma_load_2d(stage0 + i * L::kStageBytes, a_map, full0 + i * 8, (kb0 + i) * 128, m0);
          waited = true;
          s = ahead == kStages ? 0 : ahead;
          ph = ahead == kStages ? 0 : 1;
        }
#pragma unroll 2
        for (; it < n_iter; ++it) {
          alive = mbar_wait(empty0 + s * 8, ph, abort_flag, g.status, QB_DEV_WAIT_TIMEOUT_GEMM);
          if (!alive) break;
          const uint32_t fb = full0 + s * 8, st = stage0 + s * L::kStageBytes;
          mbar_arrive_expect_tx(fb, stage_tx);
          tma_load_2d(st + kBM * kRowBytes, &tmB, fb, (kb0 + it) * 128, b_row0);
          tma_load_2d(st, a_map, fb, (kb0 + it) * 128, m0);
          if (++s == kStages) { s = 0; ph ^= 1; }
        }
      }
      // s is the stage that was filled longest ago, and ph the parity of what it waits for, be it the end of the fill or its release; one
      // that was never filled passes at once.
      if (alive && *abort_flag == 0) {
        // Tail: see the last stage releases land before the CTA can exit.
        int ts = s;
        uint32_t tph = ph;
        for (int i = 0; i < kStages; ++i) {
          if (!mbar_wait(empty0 + ts * 8, tph, abort_flag, g.status, QB_DEV_WAIT_TIMEOUT_GEMM)) break;
          if (++ts == kStages) { ts = 0; tph ^= 1; }
        }
      }
      if (*abort_flag) {
        // Giving up: let the copies already in flight land before this CTA's memory goes away.
        for (int i = 0; i < kStages; ++i) {
          mbar_wait(full0 + s * 8, ph, drain_flag, g.status, QB_DEV_WAIT_TIMEOUT_GEMM);
          if (++s == kStages) { s = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer: one block of K into one buffer
    if (elect_one()) {
      const uint32_t full0 = smem_u32(full_bar), empty0 = smem_u32(empty_bar), taken0 = smem_u32(acc_empty);
      const uint64_t desc0 = umma_desc_k_sw128(smem_u32(smem));
      int s = 0;
      uint32_t ph = 0, bph = ~0u;  // bit b: parity to wait for at buffer b (a fresh one passes for parity 1); a tile begins with buffer 0
      bool landed = false, taken = false;  // what the barriers of this stage and buffer said a block earlier
      bool alive = true;
      for (int t = blockIdx.x; t < g.n_tiles && alive; t += gridDim.x) {
        int m0, n0, rows, expert;
        if (!locate(t, m0, n0, rows, expert)) continue;
#pragma unroll 1
        for (int base = 0; base < n_iter && alive; base += 4) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int it = base + i;
            if (it >= n_iter) break;
            constexpr uint32_t kOne = 1;
            const int buf = i % kAccBuffers, after = (i + 1) % kAccBuffers;
            alive = (landed || mbar_wait(full0 + s * 8, ph, abort_flag, g.status, QB_DEV_WAIT_TIMEOUT_GEMM)) &&
                    (taken || mbar_wait(taken0 + buf * 8, bph >> buf & 1, abort_flag, g.status, QB_DEV_WAIT_TIMEOUT_GEMM));
            if (!alive) break;
            tc_fence_after();
            const uint64_t a_desc = desc0 + static_cast<uint64_t>(s * (L::kStageBytes >> 4)), b_desc = a_desc + (kBM * kRowBytes >> 4);
            const uint32_t release = empty0 + s * 8;
            if (++s == kStages) { s = 0; ph ^= 1; }
            bph ^= kOne << buf;
            landed = mbar_test_wait(full0 + s * 8, ph);
            taken = it + 1 < n_iter && mbar_test_wait(taken0 + after * 8, bph >> after & 1);
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_f8(tmem_base + buf * BN, a_desc + 2 * k, b_desc + 2 * k, kIdesc, k > 0 ? 1u : 0u);
            if (it == n_iter - 1 && late(t + static_cast<int>(gridDim.x) >= g.n_tiles && blockIdx.x == gridDim.x - 1 && blockIdx.z == gridDim.z - 1, abort_flag, g.status, QB_DEV_WAIT_TIMEOUT_GEMM)) {
              alive = false;  // (the products are never announced: the other warps give up as well)
              break;
            }
            umma_commit(release);
          }
        }
      }
      if (!alive || *abort_flag) {  // giving up: the MMAs in flight still read the stages and write TMEM
        umma_commit(smem_u32(drain_bar));
        mbar_wait(smem_u32(drain_bar), 0, drain_flag, g.status, QB_DEV_WAIT_TIMEOUT_GEMM);
      }
    }
  } else if (warp >= kW0) {
    // ---------------- sums and epilogue: warp w may touch TMEM lanes 32 * (w % 4) .. + 31
    if (BN == 256) setmaxnreg_inc<kWideSumRegs>();
    const int lane_grp = warp & 3, group = (warp - kW0) >> 2, et = threadIdx.x - 32 * kW0;
    const int row = lane_grp * 32 + lane;
    if (!GROUPED) grid_dep_wait();
    const int slice_rows = kBM / (clustered ? g.splits : 1), slice_row0 = clustered ? split * slice_rows : 0;  // rows this CTA finishes
    const int nb = (g.N + 127) / 128;
    int m0 = 0, n0 = 0, rows = 0;
    // The scales of this thread's row and of its columns (of 256 columns, a thread's 128 are one block's), loaded kScales blocks ahead:
    // behind the operands' traffic a load takes over 1000 clocks, as long as four blocks of 64 columns.  (Rows and blocks past the last
    // are read as the last, without a branch.)
    const float *as = nullptr, *bs = nullptr;
    float sa[kScales], sb[kScales];
    auto fetch_scales = [&](int j, int it) {
      const unsigned at = min(it, n_iter - 1);
      sa[j] = as[static_cast<size_t>(at) * static_cast<unsigned>(g.M)];
      sb[j] = bs[at];
    };
    // the first tile from t on that has tokens, with its first scales on their way; n_tiles behind the last
    auto tile_from = [&](int t) {
      for (; t < g.n_tiles; t += gridDim.x) {
        int expert;
        if (!locate(t, m0, n0, rows, expert)) continue;
        as = after_wait(args.a_scale) + static_cast<size_t>(kb0) * g.M + min(m0 + row, m0 + rows - 1);
        bs = after_wait(args.b_scale) + static_cast<size_t>(expert * nb + min(n0 / 128 + (BN == 256 ? group : 0), nb - 1)) * g.kb_total + kb0;
#pragma unroll
        for (int j = 0; j < kScales; ++j) fetch_scales(j, j);
        break;
      }
      return t;
    };
    const uint32_t tbase = tmem_base + (static_cast<uint32_t>(lane_grp * 32) << 16) + group * kCols;
    const uint32_t done0 = smem_u32(empty_bar), taken0 = smem_u32(acc_empty);
    int ws = 0;
    uint32_t wph = 0;
    auto next_block = [&]() {
      mbar_wait_warp(done0 + ws * 8, wph, abort_flag, g.status, QB_DEV_WAIT_TIMEOUT_GEMM);
      if (++ws == kStages) { ws = 0; wph ^= 1; }
      tc_fence_after();
    };
    auto release = [&](int buf) {  // its products have been read
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(taken0 + buf * 8);
    };
    for (int tile = tile_from(blockIdx.x), next; tile < g.n_tiles; tile = next) {
      const int m = m0 + row, m_last = m0 + rows - 1, n0_of = n0;
      const bool live = row < rows, busy = lane_grp * 32 < rows;  // this thread's row, any row of this warp
      const bool one_gate = g.gate == nullptr || m0 / g.rows_per_gate == m_last / g.rows_per_gate;
      // the tile's per-column vectors, and the residuals of the 8-column groups that this thread finishes for the cluster
      if (g.bias != nullptr || g.gate != nullptr) {
        asm volatile("bar.sync 2, %0;" ::"n"(kSumThreads) : "memory");  // the last tile's readers are done
        for (int j = et; j < BN; j += kSumThreads) {
          const int n = n0 + j;
          const bool in = n < g.N;
          col[BN + j] = (in && g.bias) ? bf16_bits_to_f32(g.bias[n]) : 0.f;
          col[2 * BN + j] = (in && g.gate) ? bf16_bits_to_f32(g.gate[static_cast<size_t>(m0 / g.rows_per_gate) * g.N + n]) : 0.f;
        }
      }
      uint4 pre[BN == 64 ? BN / 32 : 1][2];
      if constexpr (BN == 64) {
        if (clustered && one_gate && g.gate != nullptr) {
#pragma unroll
          for (int k = 0; k < BN / 32; ++k) {
            const int r = et / (BN / 8) + 256 / (BN / 8) * k, mm = m0 + slice_row0 + r, n = n0 + et % (BN / 8) * 8;
            pre[k][0] = make_uint4(0u, 0u, 0u, 0u);
            if (r < slice_rows && mm < g.M && n < g.N) pre[k][0] = *reinterpret_cast<const uint4*>(g.residual + static_cast<size_t>(mm) * g.N + n);
          }
        }
      }
      float2 acc[kCols / 2];
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) acc[j] = make_float2(0.f, 0.f);
      // Of a thread's columns one part is on its way from TMEM while the last one is added.  The last block's buffer is kept: the
      // sums go back there for the epilogue, while the MMAs of the next tile fill the others.
      constexpr int kPart = kCols / 2 < 32 ? kCols / 2 : 32, kParts = kCols / kPart;
      uint32_t t[2][kPart];
      next_block();
      if (busy) {
        tmem_ld(tbase, t[0]);
#pragma unroll 1
        for (int base = 0; base < n_iter; base += kScales) {
#pragma unroll
          for (int j = 0; j < kScales; ++j) {
            const int it = base + j;
            if (it >= n_iter) break;
            const uint32_t from = tbase + j % kAccBuffers * BN;
            const float s = sa[j] * sb[j];
            const float2 s2 = make_float2(s, s);
            fetch_scales(j, it + kScales);
#pragma unroll
            for (int c = 0; c < kParts; ++c) {
              tmem_wait_ld_into(t[c & 1]);
              if (c + 1 < kParts) {
                tmem_ld(from + (c + 1) * kPart, t[(c + 1) & 1]);
              } else if (it + 1 < n_iter) {
                release(j % kAccBuffers);
                next_block();
                tmem_ld(tbase + (j + 1) % kAccBuffers * BN, t[0]);
              }
#pragma unroll
              for (int q = 0; q < kPart / 2; ++q) fma2(acc[c * (kPart / 2) + q], __uint_as_float(t[c & 1][2 * q]), __uint_as_float(t[c & 1][2 * q + 1]), s2);
            }
          }
        }
      } else {
        for (int it = 1; it < n_iter; ++it) {
          release((it - 1) % kAccBuffers);
          next_block();
        }
      }
      const int last_buf = (n_iter - 1) % kAccBuffers;
      const uint32_t taddr = tbase + last_buf * BN;
      bool ok = all_of_epilogue<kSumThreads>(*abort_flag == 0);  // (and the column vectors are in place)
      next = tile_from(tile + gridDim.x);  // m0, n0 and rows are the next tile's from here on
      const bool precise = g.c_dtype != QB_BF16;
      if (clustered) {
        if constexpr (BN == 64) {
          if (ok) {
            const uint32_t dst = map_to_cta(smem_u32(smem + L::kSliceOffset), row / slice_rows);
#pragma unroll
            for (int v = 0; v < kCols / 4; ++v)
              st_dsmem_v4(dst + 16 * slice_unit<BN>(split, group * (kCols / 4) + v, row % slice_rows, slice_rows), __float_as_uint(acc[2 * v].x), __float_as_uint(acc[2 * v].y),
                          __float_as_uint(acc[2 * v + 1].x), __float_as_uint(acc[2 * v + 1].y));
          } else if (threadIdx.x == 64) {
            tell_lost<1>(lost_flag, 0, g.splits);
          }
          cluster_sync();  // every slice's share of this CTA's rows has arrived after this barrier (warps 0 and 1 join it below)
          if (ok && *lost_flag == 0) {
            const float4* parts = reinterpret_cast<const float4*>(smem + L::kSliceOffset);
            if (precise) finish_slices<BN, true>(g, parts, col, m - row, n0_of, slice_row0, slice_rows, one_gate, pre);
            else finish_slices<BN, false>(g, parts, col, m - row, n0_of, slice_row0, slice_rows, one_gate, pre);
          }
        }
      } else {
        const bool narrow = args.c_scale != nullptr;
        if (BN == 128 && narrow) {
          // A row's group of 128 results lies with two threads: values in the registers of the sums, the larger of their maxima through
          // shared memory.  (Through TMEM and 16 columns at a time, two passes of a loop, a tile took 1.8 us longer.)
          if constexpr (BN == 128) {
            float top = 0.f;
            if (ok && live) {
#pragma unroll
              for (int c = 0; c < kCols; c += 16) {
                const int n = n0_of + group * kCols + c;
                if (n < g.N) {
                  float v[16];
#pragma unroll
                  for (int q = 0; q < 8; ++q) {
                    v[2 * q] = acc[c / 2 + q].x;
                    v[2 * q + 1] = acc[c / 2 + q].y;
                  }
                  epilogue16_values<BN, true>(g, v, m, n, col + group * kCols + c, reinterpret_cast<const uint4*>(g.residual + static_cast<size_t>(m) * g.N + n), one_gate);
#pragma unroll
                  for (int q = 0; q < 8; ++q) {
                    if (q < 4 || n + 8 < g.N) top = fmaxf(top, fmaxf(fabsf(v[2 * q]), fabsf(v[2 * q + 1])));
                    acc[c / 2 + q] = make_float2(v[2 * q], v[2 * q + 1]);
                  }
                }
              }
            }
            tops[group * kBM + row] = top;
            asm volatile("bar.sync 2, %0;" ::"n"(kSumThreads) : "memory");
            if (ok && live) {
              const float s = block_scale(fmaxf(tops[row], tops[kBM + row]), args.pow2 != 0), inv = __frcp_rn(s);
              if (group == 0) args.c_scale[static_cast<size_t>(n0_of / 128) * g.M + m] = s;
              uint8_t* c_row = static_cast<uint8_t*>(g.C) + static_cast<size_t>(m) * g.N;
#pragma unroll
              for (int c = 0; c < kCols; c += 16) {
                const int n = n0_of + group * kCols + c;
                uint32_t w[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  const float2 x = acc[c / 2 + 2 * q], y = acc[c / 2 + 2 * q + 1];
                  w[q] = pack_e4m3x4(__fmul_rn(x.x, inv), __fmul_rn(x.y, inv), __fmul_rn(y.x, inv), __fmul_rn(y.y, inv));
                }
                if (n >= g.N) continue;
                if (g.N % 16 == 0) {
                  *reinterpret_cast<uint4*>(c_row + n) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                  *reinterpret_cast<uint2*>(c_row + n) = make_uint2(w[0], w[1]);
                  if (n + 8 < g.N) *reinterpret_cast<uint2*>(c_row + n + 8) = make_uint2(w[2], w[3]);
                }
              }
            }
          }
        } else if (ok && busy) {
          float row_top = 0.f;
          // (a warp reads back what it wrote itself)
#pragma unroll
          for (int c = 0; c < kParts; ++c) {
#pragma unroll
            for (int q = 0; q < kPart / 2; ++q) {
              t[c & 1][2 * q] = __float_as_uint(acc[c * (kPart / 2) + q].x);
              t[c & 1][2 * q + 1] = __float_as_uint(acc[c * (kPart / 2) + q].y);
            }
            tmem_st(taddr + c * kPart, t[c & 1]);
          }
          tmem_wait_st();
          const bool wide = g.N % 32 == 0 && (reinterpret_cast<uintptr_t>(g.C) & 31u) == 0;
          uint8_t* c_row = live ? row_of_c(g, m) : nullptr;
          const uint4* res_row = reinterpret_cast<const uint4*>(g.residual + static_cast<size_t>(m) * g.N + n0_of);
          const int c0 = group * kCols;
          uint4 coming[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};  // residual of the next turn
          auto fetch = [&](int c) {
            if (g.gate != nullptr && c < c0 + kCols && live && n0_of + c < g.N) {
              coming[0] = res_row[c / 8];
              if (n0_of + c + 8 < g.N) coming[1] = res_row[c / 8 + 1];
            }
          };
          fetch(c0);
          float top = 0.f;
#pragma unroll 1
          for (int c = c0; c < c0 + kCols; c += 16) {
            if (n0_of + c >= g.N) break;
            uint4 res[2] = {coming[0], coming[1]};
            uint32_t r[16];
            tmem_ld16(taddr + c - c0, r);
            fetch(c + 16);
            tmem_wait_ld_into(r);
            if (!narrow) {
              if (!live) continue;
              if (precise) epilogue16<BN, true>(g, r, m, n0_of + c, col + c, res, one_gate, c_row, wide, true);
              else epilogue16<BN, false>(g, r, m, n0_of + c, col + c, res, one_gate, c_row, wide, true);
            } else {
              float v[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
              if (live) epilogue16_values<BN, true>(g, v, m, n0_of + c, col + c, res, one_gate);
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                if (j < 8 || n0_of + c + 8 < g.N) top = fmaxf(top, fabsf(v[j]));
                r[j] = __float_as_uint(v[j]);
              }
              tmem_st16(taddr + c - c0, r);
            }
          }
          if (narrow) {
            tmem_wait_st();
            row_top = top;
          }
          if constexpr (BN == 256) {  // (a thread has a whole group)
            if (narrow) {
              const float s = block_scale(row_top, args.pow2 != 0), inv = __frcp_rn(s);
              const int block = n0_of / 128 + group;
              if (live && block < nb) args.c_scale[static_cast<size_t>(block) * g.M + m] = s;
              uint8_t* c_row = static_cast<uint8_t*>(g.C) + static_cast<size_t>(m) * g.N;
              const bool wide = g.N % 16 == 0;
#pragma unroll 1
              for (int c = group * kCols; c < (group + 1) * kCols; c += 16) {
                const int n = n0_of + c;
                if (n >= g.N) break;
                uint32_t r[16], w[4];
                tmem_ld16(taddr + c - group * kCols, r);
                tmem_wait_ld_into(r);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  w[j] = pack_e4m3x4(__fmul_rn(__uint_as_float(r[4 * j]), inv), __fmul_rn(__uint_as_float(r[4 * j + 1]), inv), __fmul_rn(__uint_as_float(r[4 * j + 2]), inv),
                                     __fmul_rn(__uint_as_float(r[4 * j + 3]), inv));
                if (!live) continue;
                if (wide) {
                  *reinterpret_cast<uint4*>(c_row + n) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                  *reinterpret_cast<uint2*>(c_row + n) = make_uint2(w[0], w[1]);
                  if (n + 8 < g.N) *reinterpret_cast<uint2*>(c_row + n + 8) = make_uint2(w[2], w[3]);
                }
              }
            }
          }
        }
      }
      release(last_buf);
      if (!ok) break;
    }
  }

  tc_fence_before();
  if (clustered && warp < 2) {
    __syncwarp();
    cluster_sync();  // the barrier after which the epilogue warps read what was pushed to them
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ---------------------------------------------------------------- host side
struct BlockPlan {
  int bn, splits, kb_total, kb_per_split;
};

// Width of the tiles and number of K slices.
static BlockPlan plan_blocks(const qb_gemm_blocks_params& p, int row_tiles) {
  const int kb_total = (p.K + 127) / 128, sms = num_sms();
  auto slices = [&](int s) { return (kb_total + (kb_total + s - 1) / s - 1) / ((kb_total + s - 1) / s) == s; };  // every one has a block
  const int asked = p.split_k > 1 && !slices(p.split_k) ? 1 : p.split_k;
  BlockPlan best{128, 1, kb_total, kb_total};
  double best_cost = 1e30;
  for (int bn = 64; bn <= 256; bn *= 2) {
    if (p.tile_n != 0 && p.tile_n != bn) continue;
    if (p.c_dtype == QB_E4M3 && bn == 64) continue;  // a group of 128 results is one tile's
    if (bn > 64 && p.tile_n == 0 && p.N <= bn / 2 && !(p.c_dtype == QB_E4M3 && bn == 128)) continue;
    for (int s = 1; s <= (bn == 64 ? 8 : 1); s *= 2) {
      if (asked != 0 && asked != s) continue;
      const int kbps = (kb_total + s - 1) / s;
      if (!slices(s) || (s > 1 && asked == 0 && kbps < 4)) continue;
      const long tiles = static_cast<long>(row_tiles) * ((p.N + bn - 1) / bn);
      // Measured: ns per block of K (more where the operands of over a hundred CTAs share the way out of L2), what a tile adds, and the
      // set-up of a launch.  Slices add their exchange, which grows with the CTAs that push at once.
      const long slots = s == 4 ? 33 : s == 8 ? 15 : sms / s;  // clusters that run at once (counted on a B200 of 148 SMs; the driver is not asked)
      const long rounds = (tiles + slots - 1) / slots;
      const bool busy = tiles * s > 100;
      const double per_kb = bn == 64 ? 195.0 : bn == 128 ? (busy ? 290.0 : 230.0) : (busy ? 600.0 : 530.0);
      double cost = 3500.0 + rounds * (kbps * per_kb + 600.0 + 4.0 * bn + (bn == 256 && p.c_dtype == QB_E4M3 ? 2500.0 : 0.0));
      if (s > 1) cost += 300.0 + 12.0 * tiles * s + (rounds - 1) * 4000.0;
      if (cost < best_cost) {
        best_cost = cost;
        best = BlockPlan{bn, s, kb_total, kbps};
      }
    }
  }
  return best;
}

template <int BN, bool GROUPED>
static int32_t launch_blocks(const CUtensorMap& tmA, const CUtensorMap& tmA_small, const CUtensorMap& tmB, const BlockArgs& a, dim3 grid, cudaStream_t st) {
  using L = BlockSmem<BN>;
  static std::atomic<unsigned long long> configured{0};  // one bit per device
  int dev = 0;
  QB_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= 64 || (configured.load(std::memory_order_relaxed) >> dev & 1) == 0) {
    QB_CUDA_OK(cudaFuncSetAttribute(gemm_blocks_kernel<BN, GROUPED>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kTotal));
    cudaFuncAttributes fa;
    QB_CUDA_OK(cudaFuncGetAttributes(&fa, gemm_blocks_kernel<BN, GROUPED>));
    QB_REQUIRE(BN != 256 || fa.numRegs >= kWideLaunchRegs, QB_ERR_UNSUPPORTED, "gemm_blocks: built with %d registers a thread, %d needed", fa.numRegs, kWideLaunchRegs);
    if (dev < 64) configured.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kBlockThreads<BN>);
  cfg.dynamicSmemBytes = L::kTotal;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (g_dependent_launch) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (a.g.cluster) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = 1;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = static_cast<unsigned>(a.g.splits);
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm_blocks_kernel<BN, GROUPED>, tmA, tmA_small, tmB, a);
  ++g_launch_count;
  if (e != cudaSuccess) return fail(QB_ERR_LAUNCH, "gemm kernel (block scales, %d columns, %d slices): %s", BN, a.g.splits, cudaGetErrorString(e));
  return QB_OK;
}

static int32_t validate_blocks(const qb_gemm_blocks_params* p) {
  QB_REQUIRE(p != nullptr, QB_ERR_INVALID_ARG, "gemm_blocks: params are NULL");
  QB_REQUIRE(p->M > 0 && p->N > 0 && p->K > 0, QB_ERR_INVALID_ARG, "gemm_blocks: M, N, K must be positive (got %d, %d, %d)", p->M, p->N, p->K);
  constexpr int kMost = 0x7fffffff - 255;  // rounded up to whole tiles it is still an int
  QB_REQUIRE(p->M <= kMost && p->N <= kMost && p->K <= kMost, QB_ERR_INVALID_ARG, "gemm_blocks: M, N, K too large (got %d, %d, %d)", p->M, p->N, p->K);
  QB_REQUIRE(p->c_dtype == QB_BF16 || p->c_dtype == QB_F32 || p->c_dtype == QB_E4M3, QB_ERR_INVALID_ARG, "gemm_blocks: c_dtype %d", p->c_dtype);
  QB_REQUIRE(p->K % 16 == 0, QB_ERR_ALIGN, "gemm_blocks: K = %d must be a multiple of 16", p->K);
  QB_REQUIRE(p->N % 8 == 0, QB_ERR_ALIGN, "gemm_blocks: N = %d must be a multiple of 8", p->N);
  QB_REQUIRE(p->activation == 0 || p->activation == 1, QB_ERR_INVALID_ARG, "gemm_blocks: activation %d", p->activation);
  QB_REQUIRE(p->tile_n == 0 || p->tile_n == 64 || p->tile_n == 128 || p->tile_n == 256, QB_ERR_INVALID_ARG, "gemm_blocks: tile_n %d", p->tile_n);
  QB_REQUIRE(p->split_k >= 0 && p->split_k <= 8 && (p->split_k & (p->split_k - 1)) == 0, QB_ERR_INVALID_ARG, "gemm_blocks: split_k %d", p->split_k);
  const bool wide = p->c_dtype == QB_E4M3 || p->tile_n > 64;  // (a group of 128 results is one tile's)
  QB_REQUIRE(p->split_k <= 1 || !wide, QB_ERR_UNSUPPORTED, "gemm_blocks: K slices go with tiles of 64 columns and a bf16 or f32 result");
  QB_REQUIRE(p->tile_n != 64 || !wide, QB_ERR_UNSUPPORTED, "gemm_blocks: an e4m3 result goes with tiles of 128 or 256 columns");
  return QB_OK;
}

static int32_t blocks_run(const void* A, const void* B, const float* a_scale, const float* b_scale, void* C, float* c_scale, const void* bias, const void* gate,
                          const void* residual, const int* tile_expert, const int* tile_rows, int n_experts, const qb_gemm_blocks_params* p, cudaStream_t st) {
  int32_t rc = validate_blocks(p);
  if (rc != QB_OK) return rc;
  QB_REQUIRE(A && B && C && a_scale && b_scale, QB_ERR_INVALID_ARG, "gemm_blocks: A, B, C and the scales must not be NULL");
  QB_REQUIRE((gate == nullptr) == (residual == nullptr), QB_ERR_INVALID_ARG, "gemm_blocks: gate and residual come together");
  QB_REQUIRE((c_scale != nullptr) == (p->c_dtype == QB_E4M3), QB_ERR_INVALID_ARG, "gemm_blocks: an e4m3 C has scales, another has none");
  QB_REQUIRE(aligned16(A) && aligned16(B) && aligned16(C) && aligned16(bias) && aligned16(gate) && aligned16(residual), QB_ERR_ALIGN,
             "gemm_blocks: every matrix must be 16-byte aligned");
  QB_REQUIRE(((reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(b_scale) | reinterpret_cast<uintptr_t>(c_scale)) & 3u) == 0, QB_ERR_ALIGN,
             "gemm_blocks: scales must be 4-byte aligned");
  unsigned int* status = status_word();
  QB_REQUIRE(status != nullptr, QB_ERR_CUDA, "gemm_blocks: device status word unavailable");
  const bool grouped = tile_expert != nullptr;
  BlockArgs a{};
  GemmArgs& g = a.g;
  g.rows_per_gate = p->M;
  if (gate != nullptr) {
    QB_REQUIRE(p->gate_groups >= 1 && p->M % p->gate_groups == 0, QB_ERR_INVALID_ARG, "gemm_blocks: gate_groups %d does not divide M = %d", p->gate_groups, p->M);
    g.rows_per_gate = p->M / p->gate_groups;
  }
  const int row_tiles = (p->M + kBM - 1) / kBM;
  // Grouped: the slots are what any routing fits; with few tokens an expert's run is one tile, with many it ends halfway in one.
  const int used_tiles = !grouped ? row_tiles : 2 * row_tiles <= 3 * n_experts ? (row_tiles < n_experts ? row_tiles : n_experts) : row_tiles - n_experts / 2;
  const BlockPlan pl = plan_blocks(*p, used_tiles);
  g.M = p->M; g.N = p->N; g.K = p->K;
  g.a_rows = p->M < kBM ? (p->M + 7) / 8 * 8 : kBM;
  g.kb_total = pl.kb_total; g.kb_per_split = pl.kb_per_split; g.splits = pl.splits; g.cluster = pl.splits > 1;
  g.b_const = p->b_constant != 0;
  g.c_dtype = p->c_dtype; g.activation = p->activation;
  g.bias = static_cast<const uint16_t*>(bias);
  g.gate = static_cast<const uint16_t*>(gate);
  g.residual = static_cast<const uint16_t*>(residual);
  g.C = C;
  g.status = status;
  g.tile_expert = tile_expert;
  a.a_scale = a_scale; a.b_scale = b_scale; a.c_scale = c_scale; a.tile_rows = tile_rows; a.pow2 = p->pow2 != 0; a.n_experts = n_experts;
  a.small_rows = grouped ? 32 : 0;
  CUtensorMap tmA, tmA_small, tmB;
  rc = make_tmap_2d_sw(&tmA, A, 1, p->M, p->K, g.a_rows, 128, 128);
  if (rc != QB_OK) return rc;
  tmA_small = tmA;
  if (grouped) {
    rc = make_tmap_2d_sw(&tmA_small, A, 1, p->M, p->K, a.small_rows, 128, 128);
    if (rc != QB_OK) return rc;
  }
  rc = make_tmap_2d_sw(&tmB, B, 1, static_cast<uint64_t>(p->N) * n_experts, p->K, pl.bn, 128, 128);
  if (rc != QB_OK) return rc;
  g.tiles_m = row_tiles;
  const long long n_tiles = static_cast<long long>(row_tiles) * ((p->N + pl.bn - 1) / pl.bn);
  QB_REQUIRE(n_tiles < (1ll << 30), QB_ERR_INVALID_ARG, "gemm_blocks: %lld tiles", n_tiles);
  g.n_tiles = static_cast<int>(n_tiles);
  const dim3 grid(pl.splits > 1 || n_tiles < num_sms() ? g.n_tiles : num_sms(), 1, pl.splits);
  if (grouped) return pl.bn == 256 ? launch_blocks<256, true>(tmA, tmA_small, tmB, a, grid, st) : pl.bn == 128 ? launch_blocks<128, true>(tmA, tmA_small, tmB, a, grid, st) : launch_blocks<64, true>(tmA, tmA_small, tmB, a, grid, st);
  return pl.bn == 256 ? launch_blocks<256, false>(tmA, tmA_small, tmB, a, grid, st) : pl.bn == 128 ? launch_blocks<128, false>(tmA, tmA_small, tmB, a, grid, st) : launch_blocks<64, false>(tmA, tmA_small, tmB, a, grid, st);
}

}  // namespace qb

using namespace qb;

extern "C" int32_t qb_gemm_blocks(const void* A, const void* B, const float* a_scale, const float* b_scale, void* C, float* c_scale, const void* bias, const void* gate,
                                  const void* residual, const qb_gemm_blocks_params* p, void* stream) {
  return blocks_run(A, B, a_scale, b_scale, C, c_scale, bias, gate, residual, nullptr, nullptr, 1, p, static_cast<cudaStream_t>(stream));
}

extern "C" int32_t qb_gemm_grouped_blocks(const void* A, const void* B, const float* a_scale, const float* b_scale, void* C, float* c_scale, const int32_t* tile_expert,
                                          const int32_t* tile_rows, int32_t n_experts, const qb_gemm_blocks_params* p, void* stream) {
  QB_REQUIRE(p != nullptr && tile_expert != nullptr && tile_rows != nullptr, QB_ERR_INVALID_ARG, "gemm_grouped_blocks: params or tile tables are NULL");
  QB_REQUIRE(p->M > 0 && p->M % kBM == 0, QB_ERR_UNSUPPORTED, "gemm_grouped_blocks: M = %d must be a multiple of 128", p->M);
  QB_REQUIRE(n_experts >= 1 && static_cast<long long>(n_experts) * p->N < (1ll << 31), QB_ERR_INVALID_ARG, "gemm_grouped_blocks: %d experts", n_experts);
  QB_REQUIRE(p->split_k <= 1, QB_ERR_UNSUPPORTED, "gemm_grouped_blocks: split_k %d", p->split_k);
  qb_gemm_blocks_params q = *p;
  q.split_k = 1;  // a padding tile leaves before any K slice could wait for it
  return blocks_run(A, B, a_scale, b_scale, C, c_scale, nullptr, nullptr, nullptr, tile_expert, tile_rows, n_experts, &q, static_cast<cudaStream_t>(stream));
}
