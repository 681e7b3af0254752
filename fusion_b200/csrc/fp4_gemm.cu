// Grouped expert product of microscaled 4-bit rows on the block-scaled tensor cores.
//
//   out[r, n] = gw_e gx row_scale_r sum_k (qw sw)[e, n, k] (qx sx)[r, k]
//   SwiGLU: out[r, f] = silu(y[r, f]) y[r, I + f]
//
// tcgen05.mma kind::mxf4nvf4 (NV, scale_vec::4X) / kind::mxf4 (MX, scale_vec::2X) multiplies
// 4-bit operands from shared memory with their scales from tensor memory and accumulates in
// fp32 there, so nothing is expanded: a weight costs 0.56 or 0.53 bytes from HBM and the
// product runs at four times the bf16 rate. The weights are the M side (128 rows), the tokens
// of one dispatch block the N side (16..256), as in the bf16 grouped GEMM: one token still
// streams weights through full-width tiles.
//
// A CTA loops over (block, weight tile) units with one continuous ring of stages (256 K
// elements = 128 bytes of a row):
//   warp 0  : producer, one lane: a TMA box of weights and one of token rows (128-byte swizzle),
//             one bulk copy each of their scale atoms
//   warp 1  : TMEM owner; one lane issues a stage's four K = 64 MMAs
//   warp 2  : one lane copies a stage's scales into tensor memory (tcgen05.cp) ahead of the
//             MMAs, into columns of that stage. Issued by the MMA thread they would run in order
//             with the MMAs, about 55 cycles each: 12 of them for 512 cycles of MMA (dense
//             8192 x 4096 x 6144 NV: 290 -> 230 us with 128-token blocks)
//   warps 4-7: epilogue, TMEM -> registers -> shared (token-major) -> 16-byte stores
// The accumulator is double-buffered: the next unit's MMAs run while the epilogue drains.
// Blocks up to 64 tokens run here, two CTAs on an SM (bound by HBM: the weights); wider ones on
// SM pairs, fp4_gemm_pair.cuh.
#include "fp4.cuh"
#include "host_util.h"

namespace fus {
namespace {

struct Fp4Args {
  const uint8_t* wsf;
  const float* wg;
  const uint8_t* xsf;
  const float* xg;
  const int* expert_ids;
  const int* ntp;
  const int* live_ids;
  int live_limit;
  int x_rows;
  int n_experts;
  int w_rows;
  int out_cols;
  int K;
  int nst;      // stages along K
  int m_tiles;  // weight tiles of an expert
  int scatter;
  int out_f32;
  int stream_w;  // each weight tile meets one token block
  const float* row_scale;
  void* out;
  long ldo;
  int out_rows;
  int pdl;
  int* status;
};

// The rows of a token block in one box: the smallest of these maps that holds the live ones
// (32, 64, 96 or 128 rows; blocks up to 64 rows use the first, with a box of the block). A
// copy costs about 75 cycles beside its bytes, so one is issued, not four of 32 rows (copies
// alone, 8192 x 4096 x 6144 by pairs: 92 -> 72 us).
struct TokenMaps {
  CUtensorMap m[4];
};

constexpr long kSpreadElements = 1 << 22;  // see fus_fp4_expert_gemm

constexpr int kGroupThreads = 128;  // an epilogue group: the four lane quarters of TMEM

template <int BN, int FMT>
struct Cfg {
  static constexpr int CELLS = fp4_cells(FMT);
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = BN * 128;
  static constexpr int SFA_BYTES = CELLS * 512;
  static constexpr int SFB_BYTES = CELLS * 512;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;
  static constexpr int CHUNK = BN < 32 ? BN : 32;  // token columns of an epilogue step
  static constexpr int THREADS = 128 + kGroupThreads;
  static constexpr int EPI_BYTES = CHUNK * 128 * 4 + BN * 4;  // staging, row numbers
  static constexpr int CTAS = 2;                              // for an SM (TMEM 256 columns each)
  static constexpr int RING_TARGET = 112 * 1024 - EPI_BYTES - 1280;
  static constexpr int STAGES = RING_TARGET / STAGE_BYTES > 8 ? 8 : RING_TARGET / STAGE_BYTES;
  static constexpr int ACCS = 2;
  static constexpr int SFB_OFF = CELLS * 4;                      // token scales, after the weights'
  static constexpr int SF_COLS = SFB_OFF + CELLS * 4;            // a stage's scales
  static constexpr int SF_COL = ACCS * BN;
  static constexpr int COLS = SF_COL + STAGES * SF_COLS;
  static constexpr int TMEM_COLS = COLS <= 128 ? 128 : 256;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_BYTES + 256 + 1024;
  static_assert(STAGES >= 3 && CTAS * TMEM_COLS <= 512 && COLS <= TMEM_COLS, "resources");
};

// Instruction descriptor of the block-scaled kinds: bits 4-5 B scale id, 7-9 / 10-11 A / B
// type (1 = e2m1), 17-22 N >> 3, 23 scale type (1 = e8m0, 0 = e4m3), 24-28 M >> 4, 29-30 A
// scale id (which bytes of the 32-bit scale cell this MMA reads: 0 or 2 for scale_vec::2X)
template <int FMT>
FUS_DEVICE uint32_t fp4_idesc(int m, int n, int id) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) |
         ((FMT == FUS_FP4_MX ? 1u : 0u) << 23) | ((uint32_t)(m >> 4) << 24) |
         ((uint32_t)id << 4) | ((uint32_t)id << 29);
}

template <int FMT>
FUS_DEVICE void tc_mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                           uint32_t sfb, uint32_t accumulate) {
  if (FMT == FUS_FP4_MX)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], "
        "[%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, "
        "[%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// one 512-byte scale atom in shared memory: no swizzle, 8-row core matrices of 128 bytes
// following one another
FUS_DEVICE uint64_t scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3fff) | ((uint64_t)8 << 16) | ((uint64_t)8 << 32) |
         ((uint64_t)1 << 46);
}
// ... into tensor memory (4 columns, repeated over the 4 lane quarters)
FUS_DEVICE void tc_cp_scales(uint32_t taddr, uint32_t saddr) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr),
               "l"(scale_desc(saddr))
               : "memory");
}

// The group's staged chunk, token-major [CHUNK][128] fp32, to its output rows: nj live tokens,
// rows[] their output rows (-1: none), weight tile mt; 16 bytes for a thread and row.
template <bool SWIGLU, int CHUNK>
FUS_DEVICE void store_chunk(const Fp4Args& a, const float* S, const int* rows, int nj, int mt,
                            int et) {
  constexpr int PER = SWIGLU ? 8 : 16;  // threads of a token row, 8 features each
  const int f = (et % PER) * 8;
  const int col = mt * (SWIGLU ? 64 : 128) + f;
#pragma unroll
  for (int j0 = 0; j0 < CHUNK; j0 += kGroupThreads / PER) {
    const int j = j0 + et / PER;
    if (j >= nj || col >= a.out_cols) continue;
    const int row = rows[j];
    if (row < 0) continue;
    float o[8];
    *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(S + j * 128 + f);
    *reinterpret_cast<float4*>(o + 4) = *reinterpret_cast<const float4*>(S + j * 128 + f + 4);
    if (SWIGLU) {
      float w[8];
      *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(S + j * 128 + 64 + f);
      *reinterpret_cast<float4*>(w + 4) = *reinterpret_cast<const float4*>(S + j * 128 + 68 + f);
#pragma unroll
      for (int t = 0; t < 8; ++t) o[t] = silu_mul(o[t], w[t]);
    }
    if (a.row_scale) {
      const float rs = __ldg(a.row_scale + row);
#pragma unroll
      for (int t = 0; t < 8; ++t) o[t] *= rs;
    }
    if (a.out_f32) {
      float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + (long)row * a.ldo + col);
      d[0] = make_float4(o[0], o[1], o[2], o[3]);
      d[1] = make_float4(o[4], o[5], o[6], o[7]);
    } else {
      *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(a.out) + (long)row * a.ldo + col) =
          pack8(o);
    }
  }
}

template <int BN, int FMT, bool SWIGLU>
__global__ void __launch_bounds__((Cfg<BN, FMT>::THREADS), (Cfg<BN, FMT>::CTAS))
    fp4_gemm_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx,
                    const __grid_constant__ Fp4Args a) {
  using C = Cfg<BN, FMT>;
  constexpr int STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  const uint32_t sA = smem_u32(smem);
  const uint32_t sB = sA + STAGES * C::A_BYTES;
  const uint32_t sSA = sB + STAGES * C::B_BYTES;
  const uint32_t sSB = sSA + STAGES * C::SFA_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * C::STAGE_BYTES + C::EPI_BYTES);
  const uint32_t bar_full = smem_u32(bars);
  const uint32_t bar_empty = bar_full + 8 * STAGES;
  const uint32_t bar_acc = bar_empty + 8 * STAGES;   // accumulator finished
  const uint32_t bar_free = bar_acc + 8 * C::ACCS;   // accumulator drained
  const uint32_t bar_sf = bar_free + 8 * C::ACCS;    // a stage's scales are in tensor memory
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 3 * STAGES + 2 * C::ACCS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* group_ok = reinterpret_cast<volatile int*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
      mbar_init(bar_sf + 8 * s, 1);
    }
    for (int b = 0; b < C::ACCS; ++b) {
      mbar_init(bar_acc + 8 * b, 1);
      mbar_init(bar_free + 8 * b, 4);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tw);
    tma_prefetch_desc(&tx);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int rows_used = a.ntp ? min(__ldg(a.ntp), a.x_rows) : a.x_rows;
  const int units = (rows_used + BN - 1) / BN * a.m_tiles;
  // expert of a block; out of range: nothing of the unit is done
  auto expert_of = [&](int blk) {
    const int e = a.expert_ids ? __ldg(a.expert_ids + blk) : 0;
    if (e >= 0 && e < a.n_experts) return e;
    raise_status(a.status, FUS_ERR_BAD_EXPERT);
    return -1;
  };
  // live columns of a block (whole warp): dispatch pads end it
  auto live_of = [&](int blk) {
    int live = 0;
    for (int j = lane; j < BN; j += 32) {
      const int pos = blk * BN + j;
      live += pos < rows_used && (!a.live_ids || __ldg(a.live_ids + pos) < a.live_limit);
    }
    return __reduce_add_sync(0xffffffffu, live);
  };

  if (warp == 0) {
    const uint64_t pol_w = a.stream_w ? policy_evict_first() : policy_evict_normal();
    const uint64_t pol_x = policy_evict_last();
    int it = 0;  // stages issued
    bool waited = a.pdl == 0;
    bool ok = true;
    for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
      const int blk = u / a.m_tiles, mt = u - blk * a.m_tiles;
      const int e = expert_of(blk);
      if (e < 0) continue;
      const uint8_t* wsf = a.wsf + ((long)e * a.m_tiles + mt) * a.nst * C::SFA_BYTES;
      const uint8_t* xsf = a.xsf + (long)blk * a.nst * C::SFB_BYTES;
      auto load_w = [&](int s, int k) {
        const uint32_t full = bar_full + 8 * s;
        mbar_arrive_expect_tx(full, C::STAGE_BYTES);
        if (SWIGLU) {  // 64 gate rows, their 64 up rows
          tma_load_3d(sA + s * C::A_BYTES, &tw, full, k * 128, e * a.w_rows + mt * 64, 0, pol_w);
        } else {
          tma_load_2d(sA + s * C::A_BYTES, &tw, full, k * 128, e * a.w_rows + mt * 128, pol_w);
        }
        bulk_load(sSA + s * C::SFA_BYTES, wsf + (long)k * C::SFA_BYTES, C::SFA_BYTES, full, pol_w);
      };
      auto load_x = [&](int s, int k) {
        const uint32_t full = bar_full + 8 * s;
        tma_load_2d(sB + s * C::B_BYTES, &tx, full, k * 128, blk * BN, pol_x);
        bulk_load(sSB + s * C::SFB_BYTES, xsf + (long)k * C::SFB_BYTES, C::SFB_BYTES, full, pol_x);
      };
      int k0 = 0;
      if (!waited) {
        // programmatic dependent of the quantiser: the first ring's weights are requested
        // while it runs, its rows after it
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
  } else if (warp == 1) {
    int it = 0, n = 0;
    bool ok = true;
    for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
      const int blk = u / a.m_tiles;
      if (expert_of(blk) < 0) continue;
      const int nm = max(16, (live_of(blk) + 15) & ~15);
      const int buf = n % C::ACCS;
      ok = warp_wait_bounded(bar_free + 8 * buf, ((n / C::ACCS) & 1) ^ 1, abort_flag, a.status);
      tc_fence_after();
      const uint32_t acc = tmem + buf * BN;
      for (int k = 0; k < a.nst && ok; ++k, ++it) {
        const int s = it % STAGES;
        ok = warp_wait_bounded(bar_full + 8 * s, (it / STAGES) & 1, abort_flag, a.status) &&
             warp_wait_bounded(bar_sf + 8 * s, (it / STAGES) & 1, abort_flag, a.status);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t sf = tmem + C::SF_COL + s * C::SF_COLS;
          const int steps = min(4, (a.K - k * kFp4StageK + 63) / 64);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j < steps) {
              const int cell = FMT == FUS_FP4_MX ? j / 2 : j;
              const int id = FMT == FUS_FP4_MX ? (j % 2) * 2 : 0;
              tc_mma_fp4<FMT>(acc, sw128_desc(sA + s * C::A_BYTES + 32 * j),
                              sw128_desc(sB + s * C::B_BYTES + 32 * j), fp4_idesc<FMT>(128, nm, id),
                              sf + 4 * cell, sf + C::SFB_OFF + 4 * cell, (k | j) != 0);
            }
          }
          tc_commit(bar_empty + 8 * s);
          if (k == a.nst - 1) tc_commit(bar_acc + 8 * buf);
        }
        __syncwarp();
      }
      ++n;
    }
  } else if (warp == 2) {
    int it = 0;
    bool ok = true;
    for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
      const int blk = u / a.m_tiles;
      if (expert_of(blk) < 0) continue;
      for (int k = 0; k < a.nst; ++k, ++it) {
        const int s = it % STAGES;
        // a full stage: the MMAs that read its scale columns before are done
        ok = warp_wait_bounded(bar_full + 8 * s, (it / STAGES) & 1, abort_flag, a.status);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t sf = tmem + C::SF_COL + s * C::SF_COLS;
#pragma unroll
          for (int c = 0; c < C::CELLS; ++c) {
            tc_cp_scales(sf + 4 * c, sSA + s * C::SFA_BYTES + 512 * c);
            tc_cp_scales(sf + C::SFB_OFF + 4 * c, sSB + s * C::SFB_BYTES + 512 * c);
          }
          tc_commit(bar_sf + 8 * s);
        }
        __syncwarp();
      }
    }
  } else if (warp >= 4) {
    const int q4 = warp & 3;  // the TMEM lanes this warp may read
    const int m = q4 * 32 + lane;
    const int et = threadIdx.x - 128;
    float* S = reinterpret_cast<float*>(smem + STAGES * C::STAGE_BYTES);
    int* s_row = reinterpret_cast<int*>(smem + STAGES * C::STAGE_BYTES + C::CHUNK * 128 * 4);
    const float gx = a.xg ? __ldg(a.xg) : 1.0f;
    int n = 0;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      const int blk = u / a.m_tiles, mt = u - blk * a.m_tiles;
      const int e = expert_of(blk);
      if (e < 0) continue;
      const int live = live_of(blk);
      // output rows, out of range: -1 (read after the barrier below)
      for (int j = et; j < live; j += kGroupThreads) {
        const int pos = blk * BN + j;
        const int row = a.scatter ? __ldg(a.live_ids + pos) : pos;
        s_row[j] = row < a.out_rows ? row : -1;
      }
      const float alpha = (a.wg ? __ldg(a.wg + e) : 1.0f) * gx;
      const int buf = n % C::ACCS;
      // one thread of the group waits, the others rest at the barrier: 256 spinning threads
      // slow the issuing warps down
      if (et == 0) *group_ok = mbar_wait_bounded(bar_acc + 8 * buf, (n / C::ACCS) & 1, abort_flag, a.status);
      named_bar_sync(1, kGroupThreads);
      if (!*group_ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + buf * BN + ((uint32_t)(q4 * 32) << 16);
      for (int c0 = 0; c0 < live; c0 += C::CHUNK) {
        uint32_t v[C::CHUNK];
#pragma unroll
        for (int c = 0; c < C::CHUNK; c += 16) tmem_ld16_issue(acc + c0 + c, v + c);
#pragma unroll
        for (int c = 0; c < C::CHUNK; c += 16) tmem_ld_wait(v + c);
#pragma unroll
        for (int j = 0; j < C::CHUNK; ++j) S[j * 128 + m] = __uint_as_float(v[j]) * alpha;
        named_bar_sync(1, kGroupThreads);
        store_chunk<SWIGLU, C::CHUNK>(a, S, s_row + c0, min(C::CHUNK, live - c0), mt, et);
        named_bar_sync(1, kGroupThreads);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_free + 8 * buf);
      ++n;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

template <int BN, int FMT, bool SWIGLU>
int launch(const CUtensorMap& tw, const TokenMaps& tx, const Fp4Args& a, long units,
           cudaStream_t st) {
  using C = Cfg<BN, FMT>;
  auto fn = fp4_gemm_kernel<BN, FMT, SWIGLU>;
  if (int rc = ensure_smem_attr((const void*)fn, C::SMEM_BYTES, "fp4_grouped_gemm")) return rc;
  const long slots = (long)num_sms() * C::CTAS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units < slots ? units : slots));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.pdl ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, tw, tx.m[0], a);
  if (e != cudaSuccess)
    return set_error(FUS_E_LAUNCH, "fp4_grouped_gemm: %s", cudaGetErrorString(e));
  return check_launch("fp4_grouped_gemm");
}

}  // namespace

#include "fp4_gemm_pair.cuh"

namespace {

template <int FMT, bool SWIGLU>
int launch_bn(int bn, const CUtensorMap& tw, const TokenMaps& tx, const fus_fp4_gemm_desc* d,
              const Fp4Args& a, long units, cudaStream_t st) {
  switch (bn) {
    case 16: return launch<16, FMT, SWIGLU>(tw, tx, a, units, st);
    case 32: return launch<32, FMT, SWIGLU>(tw, tx, a, units, st);
    case 64: return launch<64, FMT, SWIGLU>(tw, tx, a, units, st);
    case 128: return launch_pair<128, FMT, SWIGLU>(tw, tx, d, a, (int)(units / a.m_tiles), st);
    default: return launch_pair<256, FMT, SWIGLU>(tw, tx, d, a, (int)(units / a.m_tiles), st);
  }
}

int check_gemm(const fus_fp4_gemm_desc* d) {
  if (!d) return set_error(FUS_E_INVALID, "fp4_gemm: null descriptor");
  if (d->fmt != FUS_FP4_MX && d->fmt != FUS_FP4_NV)
    return set_error(FUS_E_INVALID, "fp4_gemm: unknown format %d", d->fmt);
  if (d->epilogue != FUS_EPI_BF16 && d->epilogue != FUS_EPI_SWIGLU)
    return set_error(FUS_E_INVALID, "fp4_gemm: epilogue %d not FUS_EPI_BF16 / FUS_EPI_SWIGLU",
                     d->epilogue);
  if (d->K <= 0 || d->K % 32)
    return set_error(FUS_E_INVALID, "fp4_gemm: K=%d must be a positive multiple of 32", d->K);
  if (d->w_rows <= 0 || d->w_rows % 16)
    return set_error(FUS_E_INVALID, "fp4_gemm: w_rows=%d must be a positive multiple of 16",
                     d->w_rows);
  if (d->n_experts < 1 || (long)d->n_experts * d->w_rows > 0x7fffffffL)
    return set_error(FUS_E_INVALID, "fp4_gemm: bad n_experts %d", d->n_experts);
  if (d->block_n != 16 && d->block_n != 32 && d->block_n != 64 && d->block_n != 128 &&
      d->block_n != 256)
    return set_error(FUS_E_INVALID, "fp4_gemm: block_n %d not in {16,32,64,128,256}", d->block_n);
  if (d->x_rows < 0 || d->out_rows < 0) return set_error(FUS_E_INVALID, "fp4_gemm: bad row counts");
  if (d->out_dtype != FUS_DT_BF16 && d->out_dtype != FUS_DT_F32)
    return set_error(FUS_E_INVALID, "fp4_gemm: output is FUS_DT_BF16 or FUS_DT_F32");
  if (d->x_rows == 0) return FUS_OK;
  if (!d->wq || !d->wsf || !d->xq || !d->xsf || !d->out)
    return set_error(FUS_E_INVALID, "fp4_gemm: null pointer");
  if (!aligned16(d->wq) || !aligned16(d->wsf) || !aligned16(d->xq) || !aligned16(d->xsf) ||
      d->ldxq % 16 || d->ldxq < d->K / 2)
    return set_error(FUS_E_INVALID, "fp4_gemm: operands must be 16-byte aligned");
  const int cols = d->epilogue == FUS_EPI_SWIGLU ? d->w_rows / 2 : d->w_rows;
  if (d->ldo < cols || !aligned16(d->out) || d->ldo % (d->out_dtype == FUS_DT_F32 ? 4 : 8))
    return set_error(FUS_E_INVALID, "fp4_gemm: output rows must be 16-byte aligned");
  if (d->scatter && !d->live_ids)
    return set_error(FUS_E_INVALID, "fp4_gemm: scatter needs live_ids");
  if (d->n_experts > 1 && !d->expert_ids)
    return set_error(FUS_E_INVALID, "fp4_gemm: several experts need expert_ids");
  if (d->fmt == FUS_FP4_MX && (d->wg || d->xg))
    return set_error(FUS_E_INVALID, "fp4_gemm: FUS_FP4_MX takes no factors");
  return FUS_OK;
}

int gemm_launch(const fus_fp4_gemm_desc* d, int pdl, void* stream, int* status) {
  if (int rc = check_gemm(d)) return rc;
  if (d->x_rows == 0 || d->out_rows == 0) return FUS_OK;
  const bool sw = d->epilogue == FUS_EPI_SWIGLU;
  Fp4Args a{};
  a.wsf = reinterpret_cast<const uint8_t*>(d->wsf);
  a.wg = d->wg;
  a.xsf = reinterpret_cast<const uint8_t*>(d->xsf);
  a.xg = d->xg;
  a.expert_ids = d->expert_ids;
  a.ntp = d->ntp;
  a.live_ids = d->live_ids;
  a.live_limit = d->live_limit;
  a.x_rows = d->x_rows;
  a.n_experts = d->n_experts;
  a.w_rows = d->w_rows;
  a.out_cols = sw ? d->w_rows / 2 : d->w_rows;
  a.K = d->K;
  a.nst = (int)fp4_stages(d->K);
  a.m_tiles = sw ? ceil_div(d->w_rows / 2, 64) : ceil_div(d->w_rows, 128);
  a.scatter = d->scatter;
  a.out_f32 = d->out_dtype == FUS_DT_F32;
  const int blocks = ceil_div(d->x_rows, d->block_n);
  // weights that one block of each expert reads leave L2 first; with more blocks the second
  // one finds them there
  a.stream_w = (d->live_ids ? (long)d->live_limit : (long)d->x_rows) <=
               (long)d->n_experts * d->block_n / 2;
  a.row_scale = d->row_scale;
  a.out = d->out;
  a.ldo = d->ldo;
  a.out_rows = d->out_rows;
  a.pdl = pdl;
  a.status = status;
  const long units = (long)blocks * a.m_tiles;
  if (units > 0x7fffffffL) return set_error(FUS_E_UNSUPPORTED, "fp4_gemm: too many tiles");
  CUtensorMap tw;
  TokenMaps tx;
  const uint64_t row = (uint64_t)d->K / 2, rows = (uint64_t)d->n_experts * d->w_rows;
  const uint64_t half = (uint64_t)d->w_rows / 2;
  // SwiGLU: two planes, the gate rows and the up rows of the stack
  int rc = sw ? make_tmap_u8_3d(&tw, d->wq, row, rows - half, row, 2, half * row, 128, 64, 2)
              : make_tmap_u8_2d(&tw, d->wq, row, rows, row, 128, 128);
  for (int i = 0; i < 4 && !rc; ++i)
    rc = make_tmap_u8_2d(&tx.m[i], d->xq, row, (uint64_t)d->x_rows, (uint64_t)d->ldxq, 128,
                         d->block_n <= 64 ? d->block_n : 32 * (i + 1));
  if (rc) return rc;
  cudaStream_t st = as_stream(stream);
  if (d->fmt == FUS_FP4_MX)
    return sw ? launch_bn<FUS_FP4_MX, true>(d->block_n, tw, tx, d, a, units, st)
              : launch_bn<FUS_FP4_MX, false>(d->block_n, tw, tx, d, a, units, st);
  return sw ? launch_bn<FUS_FP4_NV, true>(d->block_n, tw, tx, d, a, units, st)
            : launch_bn<FUS_FP4_NV, false>(d->block_n, tw, tx, d, a, units, st);
}

}  // namespace
}  // namespace fus

using namespace fus;

extern "C" int fus_fp4_grouped_gemm(const fus_fp4_gemm_desc* d, void* stream, int* status) {
  return gemm_launch(d, 0, stream, status);
}

extern "C" int fus_fp4_expert_gemm(const fus_fp4_gemm_desc* d, const void* x, int x_dtype,
                                   long ldx, int src_rows, int gather_div, int* pair_ws,
                                   void* stream, int* status) {
  if (int rc = check_gemm(d)) return rc;
  if (d->x_rows == 0 || d->out_rows == 0) return FUS_OK;
  if (gather_div < 0 || (gather_div > 0 && !d->live_ids))
    return set_error(FUS_E_INVALID, "fp4_expert_gemm: gathered rows need live_ids");
  if (gather_div > 0 && (long)src_rows * gather_div < d->live_limit)
    return set_error(FUS_E_INVALID, "fp4_expert_gemm: %d rows for %d pairs", src_rows, d->live_limit);
  // Large batches: a token is quantised once and written to its pairs' rows (two launches: the
  // places, then the rows). One pass over the dispatch order, which quantises a token for each
  // of its pairs, has a launch less (2.2 us) and more to compute (1.4 to 2.2 million elements a
  // us). NV, spread / one pass: 8192 pairs of 1024 tokens, K 6144 121 / 144 us with the product,
  // 1024 of 128, K 6144 91.8 / 95.8, 1024 of 128, K 2048 19.1 / 16.9.
  const bool spread = pair_ws && gather_div > 1 &&
                      ((long)d->live_limit - src_rows) * d->K >= kSpreadElements;
  // rows in dispatch order: pads are skipped by their id, gathered or not
  if (spread) {
    // the checks of fus_fp4_quantize, on no rows
    if (int rc = fus_fp4_quantize(x, x_dtype, ldx, src_rows, d->K, d->fmt, d->xg, 0, nullptr, 1, 0,
                                  nullptr, 0, d->block_n, nullptr, 0, nullptr, stream, status))
      return rc;
    if (!x || ldx < d->K || ldx > 0x7fffffffL || d->ldxq > 0x7fffffffL)
      return set_error(FUS_E_INVALID, "fp4_expert_gemm: bad source rows");
    if (int rc = fp4_quantize_spread(x, x_dtype, ldx, src_rows, d->K, d->fmt, d->xg, d->live_ids,
                                     gather_div, d->live_limit, d->ntp, d->x_rows, d->block_n,
                                     pair_ws, const_cast<void*>(d->xq), d->ldxq,
                                     const_cast<void*>(d->xsf), stream, status))
      return rc;
  } else if (int rc = fus_fp4_quantize(x, x_dtype, ldx, src_rows, d->K, d->fmt, d->xg, 0,
                                       gather_div ? d->live_ids : nullptr,
                                       gather_div ? gather_div : 1, d->live_limit, d->ntp,
                                       d->x_rows, d->block_n, const_cast<void*>(d->xq), d->ldxq,
                                       const_cast<void*>(d->xsf), stream, status)) {
    return rc;
  }
  return gemm_launch(d, 1, stream, status);
}
