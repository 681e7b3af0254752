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
//   warp 1  : TMEM owner; one lane copies a stage's scales into tensor memory (tcgen05.cp, in
//             order with the MMAs of the same thread) and issues four K = 64 MMAs. Every stage has
//             scale columns of its own: a copy never waits for the MMAs of the stage before
//   warps 2-5: epilogue, TMEM -> registers -> shared (token-major) -> 16-byte stores
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
  static constexpr int THREADS = 64 + kGroupThreads;
  static constexpr int STAGE_OUT = CHUNK * 256;  // staged bf16 rows, two buffers
  static constexpr int EPI_BYTES = 2 * STAGE_OUT + BN * 8;  // ..., row numbers and scales
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

// ---- epilogue: TMEM -> registers -> shared -> global ----
// A warp reads its 32 lanes (weight rows) as two 16-lane fragments v[2][4 NI] of NI x 8 token
// columns: a thread has rows t / 4 and t / 4 + 8 of each half, two neighbouring tokens. With
// SwiGLU those two rows are a feature's gate and up (rows come 8 gate, 8 up), so the product
// never leaves the thread. Results go to bf16 rows of tokens by transposing 8 x 8 matrix
// stores, 16-byte pieces swizzled by the token so that neither side meets a bank twice, and
// leave as 16 bytes for a thread. (Staging fp32 by feature took 4 times the shared-memory
// passes: 8192 rows x 6144 x 2048 over 32 experts 112 us against 97.) fp32 output is written
// straight from the fragments, 32 bytes of a row by eight lanes.
template <int NI>
FUS_DEVICE void read_chunk(uint32_t taddr, uint32_t* v) {
  if (NI == 4) {
    tmem_ld_16x32_issue(taddr, v);
    tmem_ld_16x32_issue(taddr + (16u << 16), v + 16);
  } else {
    tmem_ld_16x16_issue(taddr, v);
    tmem_ld_16x16_issue(taddr + (16u << 16), v + 8);
  }
}
template <int NI>
FUS_DEVICE void wait_chunk(uint32_t* v) {
  tmem_ld_wait(v);
  if (NI == 4) tmem_ld_wait(v + 16);
}

// the chunk's finished values of one thread, in place: alpha, SwiGLU, the rows' scales rs[]
// (null: none). SwiGLU leaves them in the gate's places.
template <bool SWIGLU, int NI>
FUS_DEVICE void finish_chunk(uint32_t* v, float alpha, const float* rs, int lane) {
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const float2 sc = rs ? *reinterpret_cast<const float2*>(rs + 8 * i + 2 * (lane & 3))
                         : make_float2(1.f, 1.f);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t* r = v + h * 4 * NI + 4 * i;
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(r[j]) * alpha;
      if (SWIGLU) {
        x[0] = silu_mul(x[0], x[2]);
        x[1] = silu_mul(x[1], x[3]);
      }
      if (rs) {
        x[0] *= sc.x;
        x[1] *= sc.y;
        x[2] *= sc.x;
        x[3] *= sc.y;
      }
#pragma unroll
      for (int j = 0; j < (SWIGLU ? 2 : 4); ++j) r[j] = __float_as_uint(x[j]);
    }
  }
}

FUS_DEVICE uint32_t pack_bf(uint32_t lo, uint32_t hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(__uint_as_float(lo), __uint_as_float(hi));
  return *reinterpret_cast<const uint32_t*>(&p);
}

template <bool SWIGLU, int NI>
FUS_DEVICE void stage_chunk(const uint32_t* v, uint32_t stage, int q4, int lane) {
  const int j = lane & 7, mi = lane >> 3;
  if (SWIGLU) {  // rows of 64 features: matrices (half 0, half 1) of two token blocks
#pragma unroll
    for (int i = 0; i < NI; i += 2) {
      uint32_t m[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t* r = v + (q & 1) * 4 * NI + 4 * (i + (q >> 1));
        m[q] = pack_bf(r[0], r[1]);
      }
      stmatrix_x4_trans(stage + (8 * (i + (mi >> 1)) + j) * 128 + ((q4 * 2 + (mi & 1)) ^ j) * 16, m);
    }
  } else {  // rows of 128 features: four matrices of a token block
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      uint32_t m[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t* r = v + (q >> 1) * 4 * NI + 4 * i + 2 * (q & 1);
        m[q] = pack_bf(r[0], r[1]);
      }
      stmatrix_x4_trans(stage + (8 * i + j) * 256 + ((q4 * 4 + mi) ^ j) * 16, m);
    }
  }
}

// staged rows -> output rows (rows[]: -1 none), by the group's 128 threads
template <bool SWIGLU, int NI>
FUS_DEVICE void store_chunk(const Fp4Args& a, const uint8_t* stage, const int* rows, int nj, int mt,
                            int et) {
  constexpr int PER = SWIGLU ? 8 : 16;  // 16-byte pieces of a row
  const int q = et % PER;
  const int col = mt * PER * 8 + q * 8;
  if (col >= a.out_cols) return;
#pragma unroll
  for (int j0 = 0; j0 < 8 * NI; j0 += kGroupThreads / PER) {
    const int j = j0 + et / PER;
    if (j >= nj) continue;
    const int row = rows[j];
    if (row < 0) continue;
    *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(a.out) + (long)row * a.ldo + col) =
        *reinterpret_cast<const uint4*>(stage + j * PER * 16 + (q ^ (j & 7)) * 16);
  }
}

template <bool SWIGLU, int NI>
FUS_DEVICE void store_chunk_f32(const Fp4Args& a, const uint32_t* v, const int* rows, int nj, int mt,
                                int q4, int lane) {
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = 8 * i + 2 * (lane & 3) + e;
      const int row = j < nj ? rows[j] : -1;
      if (row < 0) continue;
      float* d = reinterpret_cast<float*>(a.out) + (long)row * a.ldo;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int sub = 0; sub < (SWIGLU ? 1 : 2); ++sub) {
          const int col = SWIGLU ? mt * 64 + q4 * 16 + h * 8 + (lane >> 2)
                                 : mt * 128 + q4 * 32 + h * 16 + sub * 8 + (lane >> 2);
          if (col < a.out_cols) d[col] = __uint_as_float(v[h * 4 * NI + 4 * i + 2 * sub + e]);
        }
    }
}

// One chunk of 8 NI token columns whose fragments v are read: `nj` of them are live, with output
// rows rows[] and scales rs[]. `turn` alternates the two staging buffers, so one barrier of the
// group is enough: a buffer is written again only after the barrier of the chunk between.
template <bool SWIGLU, int NI>
FUS_DEVICE void write_chunk(const Fp4Args& a, uint32_t* v, float alpha, uint8_t* stage, int& turn,
                            const int* rows, const float* rs, int nj, int mt, int q4, int lane,
                            int et, int barrier) {
  finish_chunk<SWIGLU, NI>(v, alpha, a.row_scale ? rs : nullptr, lane);
  if (a.out_f32) {
    store_chunk_f32<SWIGLU, NI>(a, v, rows, nj, mt, q4, lane);
    return;
  }
  stage += turn * (8 * NI * 256);
  turn ^= 1;
  stage_chunk<SWIGLU, NI>(v, smem_u32(stage), q4, lane);
  named_bar_sync(barrier, kGroupThreads);
  store_chunk<SWIGLU, NI>(a, stage, rows, nj, mt, et);
}

// Row numbers (out of range: -1) and scales of `n` columns from dispatch position `pos0`. The caller's
// next barrier of the group makes them visible.
FUS_DEVICE void load_rows(const Fp4Args& a, int pos0, int n, int* rows, float* rs, int et) {
  for (int j = et; j < n; j += kGroupThreads) {
    int row = a.scatter ? __ldg(a.live_ids + pos0 + j) : pos0 + j;
    if (row >= a.out_rows) row = -1;
    rows[j] = row;
    if (a.row_scale) rs[j] = row >= 0 ? __ldg(a.row_scale + row) : 0.f;
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
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 2 * C::ACCS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* group_ok = reinterpret_cast<volatile int*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
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
        if (SWIGLU) {  // 8 groups of 8 gate rows and their up rows
          tma_load_4d(sA + s * C::A_BYTES, &tw, full, k * 128, 0, 0, (e * a.w_rows + mt * 64) / 8,
                      pol_w);
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
  } else if (warp >= 2) {
    const int q4 = warp & 3;  // the TMEM lanes this warp may read
    const int et = threadIdx.x - 64;
    constexpr int NI = C::CHUNK / 8;
    uint8_t* stage = smem + STAGES * C::STAGE_BYTES;
    int* s_row = reinterpret_cast<int*>(stage + 2 * C::STAGE_OUT);
    float* s_rs = reinterpret_cast<float*>(s_row + BN);
    const float gx = a.xg ? __ldg(a.xg) : 1.0f;
    int n = 0, turn = 0;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      const int blk = u / a.m_tiles, mt = u - blk * a.m_tiles;
      const int e = expert_of(blk);
      if (e < 0) continue;
      const int live = live_of(blk);
      // every thread is done with the rows of the unit before
      named_bar_sync(1, kGroupThreads);
      load_rows(a, blk * BN, live, s_row, s_rs, et);
      const float alpha = (a.wg ? __ldg(a.wg + e) : 1.0f) * gx;
      const int buf = n % C::ACCS;
      // one thread waits, the others rest at the barrier
      if (et == 0) *group_ok = mbar_wait_bounded(bar_acc + 8 * buf, (n / C::ACCS) & 1, abort_flag, a.status);
      named_bar_sync(1, kGroupThreads);
      if (!*group_ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + buf * BN + ((uint32_t)(q4 * 32) << 16);
      for (int c0 = 0; c0 < live; c0 += C::CHUNK) {
        uint32_t v[8 * NI];
        read_chunk<NI>(acc + c0, v);
        wait_chunk<NI>(v);
        write_chunk<SWIGLU, NI>(a, v, alpha, stage, turn, s_row + c0, s_rs + c0, live - c0, mt, q4,
                                lane, et, 1);
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
  if (d->x_rows < 0 || d->x_rows > kMaxRows || d->out_rows < 0)
    return set_error(FUS_E_INVALID, "fp4_gemm: bad row counts");
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
  if (units > kMaxRows) return set_error(FUS_E_UNSUPPORTED, "fp4_gemm: too many tiles");
  CUtensorMap tw;
  TokenMaps tx;
  const uint64_t row = (uint64_t)d->K / 2, rows = (uint64_t)d->n_experts * d->w_rows;
  int rc;
  if (sw) {
    // tiles of 8 gate rows, their 8 up rows, the next 8, ...: (bytes, row of 8, half, group)
    const uint64_t half = (uint64_t)d->w_rows / 2;
    const uint64_t dims[4] = {row, 8, 2, (rows - half) / 8};
    const uint64_t strides[3] = {row, half * row, 8 * row};
    const uint32_t box[4] = {128, 8, 2, 8};
    rc = make_tmap_u8(&tw, d->wq, 4, dims, strides, box);
  } else {
    rc = make_tmap_u8_2d(&tw, d->wq, row, rows, row, 128, 128);
  }
  for (int i = 0; i < (d->block_n <= 64 ? 1 : 4) && !rc; ++i)
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
  if (gather_div > 0 && ((long)src_rows * gather_div < d->live_limit ||
                         (long)src_rows * gather_div > 0x7fffffffL))
    return set_error(FUS_E_INVALID, "fp4_expert_gemm: %d rows for %d pairs", src_rows, d->live_limit);
  // No pairs: the quantiser would launch nothing, and the product, launched as its dependent, would
  // overlap whatever ran before.
  if (gather_div > 0 && d->live_limit <= 0) return FUS_OK;
  // Large batches: a token is quantised once and written to its pairs' rows (two launches: the
  // places, then the rows). One pass over the dispatch order, which quantises a token for each
  // of its pairs, has a launch less (2.2 us) and more to compute (1.4 to 2.2 million elements a
  // us). NV, spread / one pass: 8192 pairs of 1024 tokens, K 6144 121 / 144 us with the product.
  // With a narrow product (32 experts x 256 rows), called eagerly, at 2, 4 and 6 Mi saved elements,
  // 8 pairs a token: K 2048 NV 16.1 / 16.5, 18.5 / 18.6, 20.6 / 24.6 us, MX 16.3 / 15.3, 18.5 / 16.6,
  // 18.6 / 20.7; K 6144 NV 19.7 / 26.2, 21.7 / 28.8, 22.5 / 30.9, MX 18.7 / 24.8, 22.0 / 26.7,
  // 22.4 / 26.9: at K 2048 the two meet about 4 Mi. Replayed in a graph, without the host's launch,
  // spreading is ahead from 1 Mi on (K 2048 NV 10.3 / 12.8).
  const bool spread = pair_ws && gather_div > 1 &&
                      ((long)d->live_limit - src_rows) * d->K >= kSpreadElements;
  // Gathered rows skip pads by their ids. Rows that are in dispatch order already are quantised as
  // they lie, pads too: what they hold reaches no output (a token is a column of its own).
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
