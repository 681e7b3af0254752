// SM-pair form of the four-bit product for blocks of 128 and 256 tokens (tcgen05 cta_group::2).
// Included by fp4_gemm.cu.
//
// At 256 tokens for an expert the product is bound by what a stage brings into shared memory
// and the MMAs read back from it, not by the tensor pipe: a 128 x 256 tile of one CTA moves
// 54 KB for 512 cycles of MMA. A cluster of two CTAs computes 256 weight rows x 256 tokens with
// M = 256 MMAs of the leader (rank 0): CTA r stages weight tile 2 mt + r with its scales, half
// of the token rows, and the scales of all of them (each SM's tensor core scales its own rows
// against all tokens). 38 KB for 512 cycles.
//
// Both CTAs' copies complete on the leader's full barrier (tensor copies of .cta_group::2, the
// scales too; no multicast). The leader's warp 1 copies both CTAs' scales into their tensor
// memory (tcgen05.cp.cta_group::2) and issues the MMAs; commits free the stage and hand over
// the accumulators on both CTAs. 256 columns hold them, two buffers of 128-token
// blocks or one of 256: the epilogue reads its half into registers at once and frees the
// buffer before it converts and stores.
#pragma once

namespace {

template <int BN, int FMT>
struct PairCfg {
  static constexpr int CELLS = fp4_cells(FMT);
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int ATOMS = fp4_atoms(BN);
  static constexpr int B_BYTES = BN / 2 * 128;  // half of the tokens
  static constexpr int SFA_BYTES = CELLS * 512;
  static constexpr int SFB_BYTES = CELLS * ATOMS * 512;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;
  static constexpr int GROUPS = 2;
  static constexpr int COLS_THREAD = BN / GROUPS;  // accumulator columns of a thread
  static constexpr int CHUNK = 32;
  static constexpr int THREADS = 64 + GROUPS * kGroupThreads;
  static constexpr int STAGE_OUT = CHUNK * 256;  // staged bf16 rows of a group, two buffers
  static constexpr int EPI_BYTES = GROUPS * (2 * STAGE_OUT + COLS_THREAD * 8);
  static constexpr int FIT = (226 * 1024 - EPI_BYTES - 1280) / STAGE_BYTES;
  static constexpr int STAGES = FIT > 7 ? 7 : FIT;
  static constexpr int ACCS = 256 / BN;  // accumulators
  static constexpr int SFB_OFF = CELLS * 4;
  static constexpr int SF_COLS = SFB_OFF + CELLS * ATOMS * 4;  // a stage's scales
  static constexpr int SF_COL = ACCS * BN;
  static constexpr int TMEM_COLS = 512;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_BYTES + 256 + 1024;
  static_assert(SF_COL + STAGES * SF_COLS <= TMEM_COLS && STAGES >= 4, "resources");
};

template <int FMT>
FUS_DEVICE void tc_mma_fp4_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                uint32_t sfb, uint32_t accumulate) {
  if (FMT == FUS_FP4_MX)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], "
        "[%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, "
        "[%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// one scale atom of each CTA of the pair into its own tensor memory
FUS_DEVICE void tc_cp_scales_pair(uint32_t taddr, uint32_t saddr) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr),
               "l"(scale_desc(saddr))
               : "memory");
}
template <int BN, int FMT, bool SWIGLU>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__((PairCfg<BN, FMT>::THREADS), 1)
    fp4_gemm_pair_kernel(const __grid_constant__ CUtensorMap tw,
                         const __grid_constant__ TokenMaps tx,
                         const __grid_constant__ CUtensorMap twsf,
                         const __grid_constant__ CUtensorMap txsf,
                         const __grid_constant__ Fp4Args a) {
  using C = PairCfg<BN, FMT>;
  constexpr int STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  // the same offsets in both CTAs: the dynamic window starts at the same address in each
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  const uint32_t sA = smem_u32(smem);
  const uint32_t sB = sA + STAGES * C::A_BYTES;
  const uint32_t sSA = sB + STAGES * C::B_BYTES;
  const uint32_t sSB = sSA + STAGES * C::SFA_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * C::STAGE_BYTES + C::EPI_BYTES);
  const uint32_t bar_full = smem_u32(bars);          // leader's used
  const uint32_t bar_empty = bar_full + 8 * STAGES;  // both
  const uint32_t bar_acc = bar_empty + 8 * STAGES;   // both
  const uint32_t bar_free = bar_acc + 8 * C::ACCS;   // leader's used
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 2 * C::ACCS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* group_ok = reinterpret_cast<volatile int*>(tmem_slot + 2);  // [GROUPS]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < C::ACCS; ++b) {
      mbar_init(bar_acc + 8 * b, 1);
      mbar_init(bar_free + 8 * b, 2 * 4 * C::GROUPS);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tw);
    tma_prefetch_desc(&tx.m[0]);
    tma_prefetch_desc(&twsf);
    tma_prefetch_desc(&txsf);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish_pair();
  }
  // barriers initialised and TMEM allocated in both CTAs before either touches the other
  tc_fence_before();
  cluster_barrier();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int rows_used = a.ntp ? min(__ldg(a.ntp), a.x_rows) : a.x_rows;
  const int m_pairs = (a.m_tiles + 1) / 2;
  const int units = (rows_used + BN - 1) / BN * m_pairs;
  const int first = (int)cluster_id_x(), stride = (int)cluster_count_x();
  auto expert_of = [&](int blk) {
    const int e = a.expert_ids ? __ldg(a.expert_ids + blk) : 0;
    if (e >= 0 && e < a.n_experts) return e;
    raise_status(a.status, FUS_ERR_BAD_EXPERT);
    return -1;
  };
  auto live_of = [&](int blk) {
    int live = 0;
    for (int j = lane; j < BN; j += 32) {
      const int pos = blk * BN + j;
      live += pos < rows_used && (!a.live_ids || __ldg(a.live_ids + pos) < a.live_limit);
    }
    return __reduce_add_sync(0xffffffffu, live);
  };
  auto width_of = [](int live) { return max(16, (live + 15) & ~15); };

  if (warp == 0) {
    // ---- producer (both CTAs) ----
    const uint64_t pol_w = a.stream_w ? policy_evict_first() : policy_evict_normal();
    const uint64_t pol_x = policy_evict_last();
    int it = 0;
    bool waited = a.pdl == 0;
    bool ok = true;
    for (int u = first; u < units && ok; u += stride) {
      const int blk = u / m_pairs, mt = (u - blk * m_pairs) * 2 + rank;
      const int e = expert_of(blk);
      if (e < 0) continue;
      const int half = width_of(live_of(blk)) / 2;  // this CTA's token rows
      const int box = (half - 1) / 32;
      const uint32_t bytes =
          2 * (C::A_BYTES + C::SFA_BYTES + C::SFB_BYTES + 32 * (box + 1) * 128);
      // scale atoms as rows of 128 bytes; a tile past the expert's last gives no output, and
      // past the last expert's reads zeros
      const int wsf_row = (e * a.m_tiles + mt) * a.nst * (C::SFA_BYTES / 128);
      const int xsf_row = blk * a.nst * (C::SFB_BYTES / 128);
      auto load_w = [&](int s, int k) {
        const uint32_t full = cluster_map(bar_full + 8 * s, 0);
        if (leader) mbar_arrive_expect_tx(bar_full + 8 * s, bytes);
        if (SWIGLU) {
          tma_load_4d_pair(sA + s * C::A_BYTES, &tw, full, k * 128, 0, 0,
                           (e * a.w_rows + mt * 64) / 8, pol_w);
        } else {
          tma_load_2d_pair(sA + s * C::A_BYTES, &tw, full, k * 128, e * a.w_rows + mt * 128, pol_w);
        }
        tma_load_2d_pair(sSA + s * C::SFA_BYTES, &twsf, full, 0,
                         wsf_row + k * (C::SFA_BYTES / 128), pol_w);
      };
      auto load_x = [&](int s, int k) {
        const uint32_t full = cluster_map(bar_full + 8 * s, 0);
        tma_load_2d_pair(sB + s * C::B_BYTES, &tx.m[box], full, k * 128, blk * BN + rank * half,
                         pol_x);
        tma_load_2d_pair(sSB + s * C::SFB_BYTES, &txsf, full, 0,
                         xsf_row + k * (C::SFB_BYTES / 128), pol_x);
      };
      int k0 = 0;
      if (!waited) {
        // programmatic dependent of the quantiser: weights first, rows after it
        k0 = min(a.nst, STAGES);
        if (elect_one())
          for (int k = 0; k < k0; ++k) load_w(k, k);
        pdl_wait();
        if (elect_one())
          for (int k = 0; k < k0; ++k) load_x(k, k);
        __syncwarp();
        it = k0;
        waited = true;
      }
      for (int k = k0; k < a.nst; ++k, ++it) {
        const int s = it % STAGES;
        ok = warp_wait_bounded(bar_empty + 8 * s, ((it / STAGES) & 1) ^ 1, abort_flag, a.status);
        if (!ok) break;
        if (elect_one()) {
          load_w(s, k);
          load_x(s, k);
        }
        __syncwarp();
      }
    }
    if (!waited) pdl_wait();
  } else if (warp == 1 && leader) {
    // ---- MMAs ----
    int it = 0, n = 0;
    bool ok = true;
    for (int u = first; u < units && ok; u += stride) {
      const int blk = u / m_pairs;
      if (expert_of(blk) < 0) continue;
      const int live = live_of(blk), nm = width_of(live);
      // atoms of token scales that hold live rows
      const int atoms = C::ATOMS > 1 && live <= 128 ? 1 : C::ATOMS;
      const int buf = n % C::ACCS;
      ok = warp_wait_bounded(bar_free + 8 * buf, ((n / C::ACCS) & 1) ^ 1, abort_flag, a.status);
      tc_fence_after();
      for (int k = 0; k < a.nst && ok; ++k, ++it) {
        const int s = it % STAGES;
        ok = warp_wait_bounded(bar_full + 8 * s, (it / STAGES) & 1, abort_flag, a.status);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t sf = tmem + C::SF_COL + s * C::SF_COLS;
#pragma unroll
          for (int c = 0; c < C::CELLS; ++c) {
            tc_cp_scales_pair(sf + 4 * c, sSA + s * C::SFA_BYTES + 512 * c);
#pragma unroll
            for (int t = 0; t < C::ATOMS; ++t)
              if (t < atoms)
                tc_cp_scales_pair(sf + C::SFB_OFF + 4 * (c * C::ATOMS + t),
                                  sSB + s * C::SFB_BYTES + 512 * (c * C::ATOMS + t));
          }
          const int steps = min(4, (a.K - k * kFp4StageK + 63) / 64);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j < steps) {
              const int cell = FMT == FUS_FP4_MX ? j / 2 : j;
              const int id = FMT == FUS_FP4_MX ? (j % 2) * 2 : 0;
              tc_mma_fp4_pair<FMT>(tmem + buf * BN, sw128_desc(sA + s * C::A_BYTES + 32 * j),
                                   sw128_desc(sB + s * C::B_BYTES + 32 * j),
                                   fp4_idesc<FMT>(256, nm, id), sf + 4 * cell,
                                   sf + C::SFB_OFF + 4 * C::ATOMS * cell, (k | j) != 0);
            }
          }
          tc_commit_pair(bar_empty + 8 * s);
          if (k == a.nst - 1) tc_commit_pair(bar_acc + 8 * buf);
        }
        __syncwarp();
      }
      ++n;
    }
  } else if (warp >= 2) {
    // ---- epilogue (both CTAs): each group has half of the columns ----
    const int q4 = warp & 3;
    const int grp = (warp - 2) >> 2;
    const int et = threadIdx.x - 64 - grp * kGroupThreads;
    constexpr int NI = C::CHUNK / 8, NCH = C::COLS_THREAD / C::CHUNK;
    uint8_t* stage = smem + STAGES * C::STAGE_BYTES + grp * (2 * C::STAGE_OUT + C::COLS_THREAD * 8);
    int* s_row = reinterpret_cast<int*>(stage + 2 * C::STAGE_OUT);
    float* s_rs = reinterpret_cast<float*>(s_row + C::COLS_THREAD);
    volatile int* my_ok = group_ok + grp;
    const float gx = a.xg ? __ldg(a.xg) : 1.0f;
    int n = 0, turn = 0;
    for (int u = first; u < units; u += stride) {
      const int blk = u / m_pairs, mt = (u - blk * m_pairs) * 2 + rank;
      const int e = expert_of(blk);
      if (e < 0) continue;
      const int live = live_of(blk) - grp * C::COLS_THREAD;  // of this group's columns
      const int buf = n % C::ACCS;
      // every thread is done with the rows of the unit before
      named_bar_sync(1 + grp, kGroupThreads);
      load_rows(a, blk * BN + grp * C::COLS_THREAD, min(live, C::COLS_THREAD), s_row, s_rs, et);
      const float alpha = (a.wg ? __ldg(a.wg + e) : 1.0f) * gx;
      // one thread of the group waits, the others rest at the barrier
      if (et == 0) *my_ok = mbar_wait_bounded(bar_acc + 8 * buf, (n / C::ACCS) & 1, abort_flag, a.status);
      named_bar_sync(1 + grp, kGroupThreads);
      if (!*my_ok) break;
      tc_fence_after();
      uint32_t v[NCH][8 * NI];
      const uint32_t acc = tmem + buf * BN + grp * C::COLS_THREAD + ((uint32_t)(q4 * 32) << 16);
#pragma unroll
      for (int c = 0; c < NCH; ++c)
        if (c * C::CHUNK < live) read_chunk<NI>(acc + c * C::CHUNK, v[c]);
#pragma unroll
      for (int c = 0; c < NCH; ++c)
        if (c * C::CHUNK < live) wait_chunk<NI>(v[c]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(cluster_map(bar_free + 8 * buf, 0));
      ++n;
#pragma unroll
      for (int c = 0; c < NCH; ++c)
        if (c * C::CHUNK < live)
          write_chunk<SWIGLU, NI>(a, v[c], alpha, stage, turn, s_row + c * C::CHUNK,
                                  s_rs + c * C::CHUNK, live - c * C::CHUNK, mt, q4, lane, et,
                                  1 + grp);
    }
  }
  // neither CTA leaves (or frees the pair's TMEM) while the other may still signal its
  // barriers or read its shared memory
  __syncwarp();
  tc_fence_before();
  cluster_barrier();
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem, C::TMEM_COLS);
}

template <int BN, int FMT, bool SWIGLU>
int launch_pair(const CUtensorMap& tw, const TokenMaps& tx, const fus_fp4_gemm_desc* d,
                const Fp4Args& a, int blocks, cudaStream_t st) {
  using C = PairCfg<BN, FMT>;
  auto fn = fp4_gemm_pair_kernel<BN, FMT, SWIGLU>;
  if (int rc = ensure_smem_attr((const void*)fn, C::SMEM_BYTES, "fp4_grouped_gemm")) return rc;
  CUtensorMap twsf, txsf;
  const uint64_t wsf_rows = (uint64_t)a.n_experts * a.m_tiles * a.nst * (C::SFA_BYTES / 128);
  const uint64_t xsf_rows = (uint64_t)blocks * a.nst * (C::SFB_BYTES / 128);
  if (wsf_rows > 0x7fffffffu || xsf_rows > 0x7fffffffu)
    return set_error(FUS_E_UNSUPPORTED, "fp4_gemm: too many scales");
  int rc = make_tmap_u8_2d(&twsf, d->wsf, 128, wsf_rows, 128, 128, C::SFA_BYTES / 128, false);
  if (!rc) rc = make_tmap_u8_2d(&txsf, d->xsf, 128, xsf_rows, 128, 128, C::SFB_BYTES / 128, false);
  if (rc) return rc;
  const long units = (long)blocks * ((a.m_tiles + 1) / 2);
  const long pairs = num_sms() / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * (units < pairs ? units : pairs)));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.pdl ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, tw, tx, twsf, txsf, a);
  if (e != cudaSuccess)
    return set_error(FUS_E_LAUNCH, "fp4_grouped_gemm: %s", cudaGetErrorString(e));
  return check_launch("fp4_grouped_gemm");
}

}  // namespace
