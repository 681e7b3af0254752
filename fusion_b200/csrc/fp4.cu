// Quantisation to and from microscaled 4-bit floating point (formats and scale layout:
// fp4.cuh), and the packing of a checkpoint's row-major scales into scale tiles.
//
// Mathematics, for a block with largest magnitude a:
//   MX  s = 2^(floor(log2 a) - 2) (0 for a = 0), clamped to [2^-127, 2^127]
//   NV  s = e4m3(a / (6 g)), to the nearest, ties to even, at most 448
//   q = e2m1(x / s) or e2m1(x / (s g)), to the nearest, ties to even, at most 6
// Every code is the one of exact arithmetic. MX only scales by powers of two, which fp32 does
// exactly. NV divides: fp32 leaves a relative error below 2^-22, so the quotient is rounded
// twice, a little smaller and a little larger (1 -+ 2^-21), and only where the two codes
// differ (some 10^-6 of the blocks) it is decided by products of at most 31 bits in fp64.
// A block with an infinity or a NaN gets the NaN scale: the product shows it.
#include "dtype.cuh"
#include "fp4.cuh"
#include "host_util.h"

namespace fus {
namespace {

FUS_DEVICE void ld32(const void* p, uint32_t* r) {  // 32 bytes in one load, read once
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7])
               : "l"(p));
}

// 16 consecutive elements as fp32; vec: p is 32-byte aligned
template <typename T>
FUS_DEVICE void load16(const T* p, bool vec, float* f) {
  if (vec) {
    uint32_t r[8 * sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) ld32(reinterpret_cast<const char*>(p) + 32 * i, r + 8 * i);
    const T* e = reinterpret_cast<const T*>(r);
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = to_f(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = to_f(p[i]);
  }
}

// e2m1 code of x over scale s*g, decided in fp64 (all products exact)
FUS_DEVICE uint32_t code_exact(float x, double p) {
  const double a = fabs((double)x);
  uint32_t c = (a > 0.25 * p) + (a >= 0.75 * p) + (a > 1.25 * p) + (a >= 1.75 * p) +
               (a > 2.5 * p) + (a >= 3.5 * p) + (a > 5.0 * p);
  return c | (__float_as_uint(x) >> 31 << 3);
}

FUS_DEVICE uint32_t cvt2(float lo, float hi) {  // two e2m1 codes, lo in the low four bits
  return __nv_cvt_float2_to_fp4x2(make_float2(lo, hi), __NV_E2M1, cudaRoundNearest);
}

// e4m3 byte nearest to a / (6 g), ties to even
FUS_DEVICE uint32_t nv_scale(float a, float g) {
  const float t = __fdividef(a, 6.0f * g);
  constexpr float kEps = 1.0f / (1 << 21);
  const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(t - t * kEps, t + t * kEps),
                                                __NV_SATFINITE, __NV_E4M3);
  uint32_t b0 = two & 0xff, b1 = two >> 8;
  if (b0 != b1) {
    const double m = 0.5 * ((double)fp4_scale_value<FUS_FP4_NV>(b0) +
                            (double)fp4_scale_value<FUS_FP4_NV>(b1));
    const double want = m * 6.0 * (double)g;
    if ((double)a > want || ((double)a == want && (b1 & 1) == 0)) b0 = b1;
  }
  return b0;
}

// One thread quantises 16 elements; the 16 threads of a row's 256 follow one another, so the
// scale bytes of a cell sit in four (NV) or eight (MX) neighbouring lanes and leave as
// one 4-byte store. Work: blockIdx.x x threads over rows x padded K / 16.
template <typename T, int FMT>
__global__ void __launch_bounds__(256)
    fp4_quantize_kernel(const T* __restrict__ x, long ldx, int x_rows, long rows,
                        const int* __restrict__ ntp, const int* __restrict__ ids, int id_div,
                        int id_limit, int K, int per_row, const float* __restrict__ gscale,
                        long rows_per_g, int tile, uint8_t* __restrict__ q, long ldq,
                        uint8_t* __restrict__ sf, int vec, int* status) {
  pdl_allow_dependents();
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const long p = i / per_row;
  const int k = (int)(i - p * per_row) * 16;
  const long used = ntp ? min((long)__ldg(ntp), rows) : rows;
  // whole groups of 16 lanes share a row, and per_row is a multiple of 16: the shuffles
  // below never cross a row
  bool live = p < used;
  long src = p;
  if (live && ids) {
    const int id = __ldg(ids + p);
    live = id >= 0 && id < id_limit;  // dispatch pads keep what their rows held
    src = id / id_div;
    if (live && src >= x_rows) {
      raise_status(status, FUS_ERR_CAPACITY);
      live = false;
    }
  }
  float f[16];
  const bool data = live && k < K;
  if (data) {
    load16(x + src * ldx + k, vec, f);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j] = 0.f;
  }
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
  if (FMT == FUS_FP4_MX) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  const bool bad = top >= 0x7f800000u;  // infinity or NaN in the block
  uint32_t byte;
  uint32_t c[8];
  if (FMT == FUS_FP4_MX) {
    const int e = (int)(top >> 23) - 2;
    byte = e > 0 ? e : 0;
    const float inv = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte)
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = cvt2(f[2 * j] * inv, f[2 * j + 1] * inv);
    if (bad) byte = 255;
  } else {
    const float g = gscale ? __ldg(gscale + (rows_per_g ? p / rows_per_g : 0)) : 1.0f;
    byte = bad ? 0x7f : nv_scale(__uint_as_float(top), g);
    const float s = fp4_scale_value<FUS_FP4_NV>(byte);
    const float pr = s * g;
    const float inv = __frcp_rn(pr);
    if (s > 0.f && pr > 1e-30f && pr < 1e30f) {
      constexpr float kLo = 1.0f - 1.0f / (1 << 21), kHi = 1.0f + 1.0f / (1 << 21);
      const float il = inv * kLo, ih = inv * kHi;
      uint32_t differ = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        c[j] = cvt2(f[2 * j] * il, f[2 * j + 1] * il);
        differ |= c[j] ^ cvt2(f[2 * j] * ih, f[2 * j + 1] * ih);
      }
      if (differ) {
        const double pd = (double)s * (double)g;
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = code_exact(f[2 * j], pd) | code_exact(f[2 * j + 1], pd) << 4;
      }
    } else if (s > 0.f) {  // a product near fp32's ends
      const double pd = (double)s * (double)g;
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = code_exact(f[2 * j], pd) | code_exact(f[2 * j + 1], pd) << 4;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = 0;
    }
  }
  if (bad) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = 0;
  }
  if (data) {
    uint2 v;
    v.x = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
    v.y = c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24;
    *reinterpret_cast<uint2*>(q + p * ldq + k / 2) = v;
  }
  // scales: NV one byte of each lane, MX one of each lane pair
  constexpr int kLanes = FMT == FUS_FP4_MX ? 8 : 4;
  const int lane = threadIdx.x & 31;
  const int step = kLanes / 4;
  const int b0 = lane & ~(kLanes - 1);
  if (!data) byte = 0;
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) word |= __shfl_sync(0xffffffffu, byte, b0 + j * step) << (8 * j);
  if (!live) return;
  const int j0 = k / fp4_block(FMT);  // this block's scale
  if (tile == 0) {
    if (k < K && (FMT == FUS_FP4_NV || (lane & 1) == 0))
      sf[p * (K / fp4_block(FMT)) + j0] = (uint8_t)byte;
  } else if ((lane & (kLanes - 1)) == 0) {
    const long per_tile = fp4_stages(K) * fp4_stage_scale_bytes(FMT, tile);
    const int r = (int)(p % tile);
    *reinterpret_cast<uint32_t*>(sf + (p / tile) * per_tile +
                                 fp4_scale_offset(FMT, tile, r, j0 & ~3)) = word;
  }
}

template <typename T, int FMT>
__global__ void __launch_bounds__(256)
    fp4_dequantize_kernel(const uint8_t* __restrict__ q, long ldq, const uint8_t* __restrict__ sf,
                          int tile, long rows, int K, int per_row,
                          const float* __restrict__ gscale, long rows_per_g, T* __restrict__ out,
                          long ldo, int vec) {
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const long p = i / per_row;
  const int k = (int)(i - p * per_row) * 16;
  if (p >= rows || k >= K) return;
  const uint2 v = *reinterpret_cast<const uint2*>(q + p * ldq + k / 2);
  const int j0 = k / fp4_block(FMT);
  const uint32_t byte =
      tile == 0 ? sf[p * (K / fp4_block(FMT)) + j0]
                : sf[(p / tile) * (fp4_stages(K) * fp4_stage_scale_bytes(FMT, tile)) +
                     fp4_scale_offset(FMT, tile, (int)(p % tile), j0)];
  const float s = fp4_scale_value<FMT>(byte);
  const float g =
      FMT == FUS_FP4_NV && gscale ? __ldg(gscale + (rows_per_g ? p / rows_per_g : 0)) : 1.0f;
  alignas(32) T o[16];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(
        (__nv_fp4x2_storage_t)((j < 4 ? v.x >> (8 * j) : v.y >> (8 * (j - 4))) & 0xff), __NV_E2M1);
    const float2 e = __half22float2(*reinterpret_cast<const __half2*>(&h));
    // value x scale has at most 6 bits: exact; the factor rounds once, the type once
    o[2 * j] = from_f<T>(e.x * s * g);
    o[2 * j + 1] = from_f<T>(e.y * s * g);
  }
  T* dst = out + p * ldo + k;
  if (vec) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T); ++j)
      reinterpret_cast<uint4*>(dst)[j] = reinterpret_cast<const uint4*>(o)[j];
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) dst[j] = o[j];
  }
}

// row-major scales [n_experts * w_rows, K / n] -> weight scale tiles of 128 rows for each
// expert; gate_up: tile t holds gate rows [64t, 64t + 64) and their up rows
__global__ void fp4_pack_kernel(const uint8_t* __restrict__ src, int n_experts, int w_rows,
                                int tiles, int n_scales, int fmt, int gate_up, long per_tile,
                                uint8_t* __restrict__ dst, long words) {
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= words) return;
  const long byte = i * 4;
  const long t = byte / per_tile;
  const int in = (int)(byte - t * per_tile);
  const int cell = in / 512;
  const int r = (in % 512) / 16 + (in % 16) / 4 * 32;
  const int e = (int)(t / tiles), tl = (int)(t % tiles);
  int row;
  if (gate_up) {
    const int f = tl * 64 + (r & 63);
    row = f < w_rows / 2 ? f + (r >= 64 ? w_rows / 2 : 0) : w_rows;
  } else {
    row = tl * 128 + r;
  }
  uint32_t word = 0;
  if (row < w_rows) {
    const uint8_t* s = src + ((long)e * w_rows + row) * n_scales;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (cell * 4 + j < n_scales) word |= (uint32_t)s[cell * 4 + j] << (8 * j);
  }
  reinterpret_cast<uint32_t*>(dst)[i] = word;
}

bool valid_tile(int tile) {
  return tile == 16 || tile == 32 || tile == 64 || tile == 128 || tile == 256;
}

template <int FMT>
int quantize_launch(const void* x, int dtype, long ldx, int x_rows, long rows, const int* ntp,
                    const int* ids, int id_div, int id_limit, int K, const float* gscale,
                    long rows_per_g, int tile, void* q, long ldq, void* sf, cudaStream_t st,
                    int* status) {
  // rows padded to whole stages: the tail's scales are written as zeros
  const int per_row = (int)(fp4_stages(K) * (kFp4StageK / 16));
  const long n = rows * per_row;
  const long blocks = (n + 255) / 256;
  if (blocks > 0x7fffffffL) return set_error(FUS_E_UNSUPPORTED, "fp4_quantize: too many rows");
  const int vec = (reinterpret_cast<uintptr_t>(x) % 32) == 0 && (ldx * dtype_size(dtype)) % 32 == 0;
  uint8_t* qq = reinterpret_cast<uint8_t*>(q);
  uint8_t* ss = reinterpret_cast<uint8_t*>(sf);
  if (dtype == FUS_DT_BF16)
    fp4_quantize_kernel<__nv_bfloat16, FMT><<<(int)blocks, 256, 0, st>>>(
        reinterpret_cast<const __nv_bfloat16*>(x), ldx, x_rows, rows, ntp, ids, id_div, id_limit,
        K, per_row, gscale, rows_per_g, tile, qq, ldq, ss, vec, status);
  else if (dtype == FUS_DT_F16)
    fp4_quantize_kernel<__half, FMT><<<(int)blocks, 256, 0, st>>>(
        reinterpret_cast<const __half*>(x), ldx, x_rows, rows, ntp, ids, id_div, id_limit, K,
        per_row, gscale, rows_per_g, tile, qq, ldq, ss, vec, status);
  else
    fp4_quantize_kernel<float, FMT><<<(int)blocks, 256, 0, st>>>(
        reinterpret_cast<const float*>(x), ldx, x_rows, rows, ntp, ids, id_div, id_limit, K,
        per_row, gscale, rows_per_g, tile, qq, ldq, ss, vec, status);
  return check_launch("fp4_quantize");
}

template <typename T, int FMT>
void dequantize_launch(const void* q, long ldq, const void* sf, int tile, long rows, int K,
                       const float* gscale, long rows_per_g, void* out, long ldo, long blocks,
                       int per_row, cudaStream_t st) {
  const int vec = (reinterpret_cast<uintptr_t>(out) % 16) == 0 && (ldo * sizeof(T)) % 16 == 0;
  fp4_dequantize_kernel<T, FMT><<<(int)blocks, 256, 0, st>>>(
      reinterpret_cast<const uint8_t*>(q), ldq, reinterpret_cast<const uint8_t*>(sf), tile, rows,
      K, per_row, gscale, rows_per_g, reinterpret_cast<T*>(out), ldo, vec);
}

int check_common(const char* what, int fmt, int dtype, long rows, int K, int tile) {
  if (fmt != FUS_FP4_MX && fmt != FUS_FP4_NV)
    return set_error(FUS_E_INVALID, "%s: unknown format %d", what, fmt);
  if (!dtype_known(dtype))
    return set_error(FUS_E_INVALID, "%s: unknown dtype %d", what, dtype);
  if (rows < 0 || rows > 0x7fffffffL) return set_error(FUS_E_INVALID, "%s: bad row count", what);
  if (K <= 0 || K % 32)
    return set_error(FUS_E_INVALID, "%s: K=%d must be a positive multiple of 32", what, K);
  if (tile != 0 && !valid_tile(tile))
    return set_error(FUS_E_INVALID, "%s: tile %d not in {0,16,32,64,128,256}", what, tile);
  return FUS_OK;
}

}  // namespace
}  // namespace fus

using namespace fus;

extern "C" size_t fus_fp4_scale_bytes(int fmt, long rows, int K, int tile) {
  if ((fmt != FUS_FP4_MX && fmt != FUS_FP4_NV) || rows < 0 || K <= 0 || K % 32) return 0;
  if (tile == 0) return (size_t)rows * (K / fp4_block(fmt));
  if (!valid_tile(tile)) return 0;
  return (size_t)((rows + tile - 1) / tile) * fp4_stages(K) * fp4_stage_scale_bytes(fmt, tile);
}

extern "C" int fus_fp4_quantize(const void* x, int dtype, long ldx, int x_rows, int K, int fmt,
                                const float* gscale, long rows_per_g, const int* ids, int id_div,
                                int id_limit, const int* ntp, long rows, int tile, void* q,
                                long ldq, void* sf, void* stream, int* status) {
  if (int rc = check_common("fp4_quantize", fmt, dtype, rows, K, tile)) return rc;
  if (rows == 0) return FUS_OK;
  if (!x || !q || !sf) return set_error(FUS_E_INVALID, "fp4_quantize: null pointer");
  if (x_rows < 1 || ldx < K) return set_error(FUS_E_INVALID, "fp4_quantize: bad source rows");
  if (!ids && rows > x_rows)
    return set_error(FUS_E_INVALID, "fp4_quantize: %ld rows of %d", rows, x_rows);
  if (ids && (id_div < 1 || id_limit < 0))
    return set_error(FUS_E_INVALID, "fp4_quantize: bad id_div / id_limit");
  if (reinterpret_cast<uintptr_t>(x) % dtype_size(dtype))
    return set_error(FUS_E_INVALID, "fp4_quantize: misaligned source");
  if (ldq < K / 2 || ldq % 16 || !aligned16(q) || !aligned16(sf))
    return set_error(FUS_E_INVALID, "fp4_quantize: packed rows must be 16-byte aligned");
  if (rows_per_g < 0) return set_error(FUS_E_INVALID, "fp4_quantize: rows_per_g < 0");
  if (fmt == FUS_FP4_MX && gscale)
    return set_error(FUS_E_INVALID, "fp4_quantize: FUS_FP4_MX takes no factor");
  cudaStream_t st = as_stream(stream);
  return fmt == FUS_FP4_MX
             ? quantize_launch<FUS_FP4_MX>(x, dtype, ldx, x_rows, rows, ntp, ids, id_div,
                                           id_limit, K, gscale, rows_per_g, tile, q, ldq, sf, st,
                                           status)
             : quantize_launch<FUS_FP4_NV>(x, dtype, ldx, x_rows, rows, ntp, ids, id_div,
                                           id_limit, K, gscale, rows_per_g, tile, q, ldq, sf, st,
                                           status);
}

extern "C" int fus_fp4_dequantize(const void* q, long ldq, const void* sf, int fmt, int tile,
                                  long rows, int K, const float* gscale, long rows_per_g,
                                  void* out, int dtype, long ldo, void* stream, int* status) {
  (void)status;
  if (int rc = check_common("fp4_dequantize", fmt, dtype, rows, K, tile)) return rc;
  if (rows == 0) return FUS_OK;
  if (!q || !sf || !out) return set_error(FUS_E_INVALID, "fp4_dequantize: null pointer");
  if (ldq < K / 2 || ldq % 8 || reinterpret_cast<uintptr_t>(q) % 8)
    return set_error(FUS_E_INVALID, "fp4_dequantize: packed rows must be 8-byte aligned");
  if (ldo < K || reinterpret_cast<uintptr_t>(out) % dtype_size(dtype))
    return set_error(FUS_E_INVALID, "fp4_dequantize: bad output rows");
  if (rows_per_g < 0) return set_error(FUS_E_INVALID, "fp4_dequantize: rows_per_g < 0");
  if (fmt == FUS_FP4_MX && gscale)
    return set_error(FUS_E_INVALID, "fp4_dequantize: FUS_FP4_MX takes no factor");
  const int per_row = K / 16;
  const long blocks = (rows * per_row + 255) / 256;
  if (blocks > 0x7fffffffL) return set_error(FUS_E_UNSUPPORTED, "fp4_dequantize: too many rows");
  cudaStream_t st = as_stream(stream);
#define FUS_DEQ(T, F) \
  dequantize_launch<T, F>(q, ldq, sf, tile, rows, K, gscale, rows_per_g, out, ldo, blocks, per_row, st)
  if (fmt == FUS_FP4_MX) {
    if (dtype == FUS_DT_BF16) FUS_DEQ(__nv_bfloat16, FUS_FP4_MX);
    else if (dtype == FUS_DT_F16) FUS_DEQ(__half, FUS_FP4_MX);
    else FUS_DEQ(float, FUS_FP4_MX);
  } else {
    if (dtype == FUS_DT_BF16) FUS_DEQ(__nv_bfloat16, FUS_FP4_NV);
    else if (dtype == FUS_DT_F16) FUS_DEQ(__half, FUS_FP4_NV);
    else FUS_DEQ(float, FUS_FP4_NV);
  }
#undef FUS_DEQ
  return check_launch("fp4_dequantize");
}

extern "C" size_t fus_fp4_weight_scale_bytes(int fmt, int n_experts, int w_rows, int K,
                                             int gate_up) {
  if ((fmt != FUS_FP4_MX && fmt != FUS_FP4_NV) || n_experts < 1 || w_rows < 1 || K <= 0 || K % 32)
    return 0;
  const long tiles = gate_up ? (w_rows / 2 + 63) / 64 : (w_rows + 127) / 128;
  return (size_t)n_experts * tiles * fp4_stages(K) * fp4_stage_scale_bytes(fmt, 128);
}

extern "C" int fus_fp4_pack_scales(const void* scales, int fmt, int n_experts, int w_rows, int K,
                                   int gate_up, void* sf, void* stream) {
  if (fmt != FUS_FP4_MX && fmt != FUS_FP4_NV)
    return set_error(FUS_E_INVALID, "fp4_pack_scales: unknown format %d", fmt);
  if (!scales || !sf || !aligned16(sf))
    return set_error(FUS_E_INVALID, "fp4_pack_scales: null or misaligned pointer");
  if (n_experts < 1 || w_rows < 1 || K <= 0 || K % 32 || (gate_up && w_rows % 2))
    return set_error(FUS_E_INVALID, "fp4_pack_scales: bad sizes");
  const int tiles = gate_up ? (w_rows / 2 + 63) / 64 : (w_rows + 127) / 128;
  const long per_tile = fp4_stages(K) * fp4_stage_scale_bytes(fmt, 128);
  const long words = (long)n_experts * tiles * per_tile / 4;
  const long blocks = (words + 255) / 256;
  if (blocks > 0x7fffffffL) return set_error(FUS_E_UNSUPPORTED, "fp4_pack_scales: too large");
  fp4_pack_kernel<<<(int)blocks, 256, 0, as_stream(stream)>>>(
      reinterpret_cast<const uint8_t*>(scales), n_experts, w_rows, tiles, K / fp4_block(fmt), fmt,
      gate_up, per_tile, reinterpret_cast<uint8_t*>(sf), words);
  return check_launch("fp4_pack_scales");
}
