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

// 16 consecutive elements as fp32 and the largest magnitude's bits; vec: p is 32-byte aligned.
// Magnitudes compare as integers: an infinity or NaN comes out on top.
template <typename T>
FUS_DEVICE uint32_t load16(const T* p, bool vec, float* f) {
  uint32_t r[8 * sizeof(T) / 2];
  T* e = reinterpret_cast<T*>(r);
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      ld32(reinterpret_cast<const char*>(p) + 32 * i, r + 8 * i);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = to_f(e[i]);
  uint32_t top = 0;
  if (sizeof(T) == 2) {  // two 16-bit magnitudes at a time
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __vmaxu2(top, r[i] & 0x7fff7fffu);
    const uint16_t m = (uint16_t)max(top & 0xffffu, top >> 16);
    return __float_as_uint(to_f(*reinterpret_cast<const T*>(&m)));
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
  return top;
}

// eight e2m1 codes of f * m, the first in the low four bits
FUS_DEVICE uint32_t cvt8(const float* f, float m) {
  uint32_t v;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(v)
      : "f"(f[0] * m), "f"(f[1] * m), "f"(f[2] * m), "f"(f[3] * m), "f"(f[4] * m), "f"(f[5] * m),
        "f"(f[6] * m), "f"(f[7] * m));
  return v;
}

// e2m1 code of x over scale s*g, decided in fp64 (all products exact)
FUS_DEVICE uint32_t code_exact(float x, double p) {
  const double a = fabs((double)x);
  uint32_t c = (a > 0.25 * p) + (a >= 0.75 * p) + (a > 1.25 * p) + (a >= 1.75 * p) +
               (a > 2.5 * p) + (a >= 3.5 * p) + (a > 5.0 * p);
  return c | (__float_as_uint(x) >> 31 << 3);
}

// eight of them
FUS_DEVICE uint32_t code8_exact(const float* f, double p) {
  uint32_t v = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) v |= code_exact(f[j], p) << (4 * j);
  return v;
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

// One thread quantises 16 elements; blockDim (UX, 256 / UX), UX a power of two >= 16 that
// divides the row's padded K / 16, so a row's 256 elements are 16 neighbouring lanes and the
// scale bytes of a cell, in four (NV) or eight (MX) of them, leave as one 4-byte store.
// Bound: HBM (2.56 bytes an element from bf16); no index is divided, the tile is a shift.
template <typename T, int FMT>
__global__ void __launch_bounds__(256)
    fp4_quantize_kernel(const T* __restrict__ x, long ldx, int x_rows, int rows,
                        const int* __restrict__ ntp, const int* __restrict__ ids, int id_div,
                        int id_limit, int K, const float* __restrict__ gscale, int rows_per_g,
                        int tile_log2, uint8_t* __restrict__ q, long ldq,
                        uint8_t* __restrict__ sf, int vec, int* status) {
  pdl_allow_dependents();
  const int p = blockIdx.x * blockDim.y + threadIdx.y;
  const int k = (blockIdx.y * blockDim.x + threadIdx.x) * 16;
  const int used = ntp ? min(__ldg(ntp), rows) : rows;
  bool live = p < used;
  int src = p;
  if (live && ids) {
    const int id = __ldg(ids + p);
    live = id >= 0 && id < id_limit;  // dispatch pads keep what their rows held
    src = id_div > 1 ? id / id_div : id;
    if (live && src >= x_rows) {
      raise_status(status, FUS_ERR_CAPACITY);
      live = false;
    }
  }
  const bool data = live && k < K;
  float f[16];
  uint32_t top = 0;
  if (data) {
    top = load16(x + (long)src * ldx + k, vec, f);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j] = 0.f;
  }
  if (FMT == FUS_FP4_MX) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  const bool bad = top >= 0x7f800000u;  // infinity or NaN in the block
  uint32_t byte;
  uint2 c;
  if (FMT == FUS_FP4_MX) {
    const int e = (int)(top >> 23) - 2;
    byte = e > 0 ? e : 0;
    const float inv = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte)
    c = make_uint2(cvt8(f, inv), cvt8(f + 8, inv));
    if (bad) byte = 255;
  } else {
    const float g =
        gscale ? __ldg(gscale + (rows_per_g ? p / rows_per_g : 0)) : 1.0f;
    byte = bad ? 0x7f : nv_scale(__uint_as_float(top), g);
    const float s = fp4_scale_value<FUS_FP4_NV>(byte);
    const float pr = s * g;
    const float inv = __frcp_rn(pr);
    constexpr float kLo = 1.0f - 1.0f / (1 << 21), kHi = 1.0f + 1.0f / (1 << 21);
    c = make_uint2(cvt8(f, inv * kLo), cvt8(f + 8, inv * kLo));
    const uint2 up = make_uint2(cvt8(f, inv * kHi), cvt8(f + 8, inv * kHi));
    // next to a border, or a product near fp32's ends: decided in fp64
    if (c.x != up.x || c.y != up.y || !(pr > 1e-30f && pr < 1e30f)) {
      const double pd = (double)s * (double)g;
      c = s > 0.f ? make_uint2(code8_exact(f, pd), code8_exact(f + 8, pd)) : make_uint2(0, 0);
    }
  }
  if (bad) c = make_uint2(0, 0);
  if (data) *reinterpret_cast<uint2*>(q + (long)p * ldq + k / 2) = c;
  // scales: NV one byte of each lane, MX one of each lane pair; zeros past K
  constexpr int kLanes = FMT == FUS_FP4_MX ? 8 : 4;
  if (!data) byte = 0;
  uint32_t word = byte << (8 * ((threadIdx.x / (kLanes / 4)) & 3));
#pragma unroll
  for (int o = kLanes / 4; o < kLanes; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
  if (!live) return;
  const int j0 = k / fp4_block(FMT);  // this block's scale
  if (tile_log2 == 0) {
    if (k < K && (FMT == FUS_FP4_NV || (threadIdx.x & 1) == 0))
      sf[(long)p * (K / fp4_block(FMT)) + j0] = (uint8_t)byte;
  } else if ((threadIdx.x & (kLanes - 1)) == 0) {
    const int tile = 1 << tile_log2;
    const long per_tile = (long)gridDim.y * blockDim.x / 16 * fp4_stage_scale_bytes(FMT, tile);
    *reinterpret_cast<uint32_t*>(sf + (p >> tile_log2) * per_tile +
                                 fp4_scale_offset(FMT, tile, p & (tile - 1), j0 & ~3)) = word;
  }
}

FUS_DEVICE void st32(void* p, const uint32_t* r) {  // 32 bytes in one store
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// The reverse, by the same threads.
template <typename T, int FMT>
__global__ void __launch_bounds__(256)
    fp4_dequantize_kernel(const uint8_t* __restrict__ q, long ldq, const uint8_t* __restrict__ sf,
                          int tile_log2, int rows, int K, const float* __restrict__ gscale,
                          int rows_per_g, T* __restrict__ out, long ldo, int vec) {
  const int p = blockIdx.x * blockDim.y + threadIdx.y;
  const int k = (blockIdx.y * blockDim.x + threadIdx.x) * 16;
  if (p >= rows || k >= K) return;
  const uint2 v = *reinterpret_cast<const uint2*>(q + (long)p * ldq + k / 2);
  const int j0 = k / fp4_block(FMT);
  const int tile = 1 << tile_log2;
  const long per_tile = (long)gridDim.y * blockDim.x / 16 * fp4_stage_scale_bytes(FMT, tile);
  const uint32_t byte =
      tile_log2 == 0 ? sf[(long)p * (K / fp4_block(FMT)) + j0]
                     : sf[(p >> tile_log2) * per_tile +
                          fp4_scale_offset(FMT, tile, p & (tile - 1), j0)];
  const float s = fp4_scale_value<FMT>(byte);
  const float g =
      FMT == FUS_FP4_NV && gscale ? __ldg(gscale + (rows_per_g ? p / rows_per_g : 0)) : 1.0f;
  uint32_t o[8 * sizeof(T) / 2];
  T* e = reinterpret_cast<T*>(o);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(
        (__nv_fp4x2_storage_t)((j < 4 ? v.x >> (8 * j) : v.y >> (8 * (j - 4))) & 0xff), __NV_E2M1);
    const float2 w = __half22float2(*reinterpret_cast<const __half2*>(&h));
    // value x scale has at most 6 bits: exact; the factor rounds once, the type once
    e[2 * j] = from_f<T>(w.x * s * g);
    e[2 * j + 1] = from_f<T>(w.y * s * g);
  }
  T* dst = out + (long)p * ldo + k;
  if (vec) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) st32(reinterpret_cast<char*>(dst) + 32 * j, o + 8 * j);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) dst[j] = e[j];
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

int log2_of(int tile) {
  int n = 0;
  while ((1 << n) < tile) ++n;
  return n;
}

// threads over the rows, padded to whole stages of K: (UX, 256 / UX), see the kernel
void shape_of(long rows, int K, dim3& grid, dim3& block) {
  const int per_row = (int)(fp4_stages(K) * (kFp4StageK / 16));
  int ux = 16;
  while (ux < 128 && per_row % (2 * ux) == 0) ux *= 2;
  block = dim3(ux, 256 / ux);
  grid = dim3((unsigned)((rows + block.y - 1) / block.y), per_row / ux);
}

template <typename T>
int quantize_launch(const void* x, long ldx, int x_rows, long rows, const int* ntp, const int* ids,
                    int id_div, int id_limit, int K, int fmt, const float* gscale,
                    long rows_per_g, int tile, void* q, long ldq, void* sf, cudaStream_t st,
                    int* status) {
  dim3 grid, block;
  shape_of(rows, K, grid, block);
  const int vec = (reinterpret_cast<uintptr_t>(x) % 32) == 0 && (ldx * (long)sizeof(T)) % 32 == 0;
  auto fn = fmt == FUS_FP4_MX ? fp4_quantize_kernel<T, FUS_FP4_MX> : fp4_quantize_kernel<T, FUS_FP4_NV>;
  fn<<<grid, block, 0, st>>>(reinterpret_cast<const T*>(x), ldx, x_rows, (int)rows, ntp, ids, id_div,
                             id_limit, K, gscale, (int)rows_per_g, log2_of(tile),
                             reinterpret_cast<uint8_t*>(q), ldq, reinterpret_cast<uint8_t*>(sf), vec,
                             status);
  return check_launch("fp4_quantize");
}

template <typename T>
int dequantize_launch(const void* q, long ldq, const void* sf, int fmt, int tile, long rows, int K,
                      const float* gscale, long rows_per_g, void* out, long ldo, cudaStream_t st) {
  dim3 grid, block;
  shape_of(rows, K, grid, block);
  const int vec = (reinterpret_cast<uintptr_t>(out) % 32) == 0 && (ldo * (long)sizeof(T)) % 32 == 0;
  auto fn = fmt == FUS_FP4_MX ? fp4_dequantize_kernel<T, FUS_FP4_MX> : fp4_dequantize_kernel<T, FUS_FP4_NV>;
  fn<<<grid, block, 0, st>>>(reinterpret_cast<const uint8_t*>(q), ldq,
                             reinterpret_cast<const uint8_t*>(sf), log2_of(tile), (int)rows, K, gscale,
                             (int)rows_per_g, reinterpret_cast<T*>(out), ldo, vec);
  return check_launch("fp4_dequantize");
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
  if (rows_per_g < 0 || rows_per_g > 0x7fffffffL) return set_error(FUS_E_INVALID, "fp4_quantize: bad rows_per_g");
  if (fmt == FUS_FP4_MX && gscale)
    return set_error(FUS_E_INVALID, "fp4_quantize: FUS_FP4_MX takes no factor");
  cudaStream_t st = as_stream(stream);
#define FUS_Q(T)                                                                               \
  quantize_launch<T>(x, ldx, x_rows, rows, ntp, ids, id_div, id_limit, K, fmt, gscale,          \
                     rows_per_g, tile, q, ldq, sf, st, status)
  if (dtype == FUS_DT_BF16) return FUS_Q(__nv_bfloat16);
  if (dtype == FUS_DT_F16) return FUS_Q(__half);
  return FUS_Q(float);
#undef FUS_Q
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
  if (rows_per_g < 0 || rows_per_g > 0x7fffffffL) return set_error(FUS_E_INVALID, "fp4_dequantize: bad rows_per_g");
  if (fmt == FUS_FP4_MX && gscale)
    return set_error(FUS_E_INVALID, "fp4_dequantize: FUS_FP4_MX takes no factor");
  cudaStream_t st = as_stream(stream);
#define FUS_D(T) \
  dequantize_launch<T>(q, ldq, sf, fmt, tile, rows, K, gscale, rows_per_g, out, ldo, st)
  if (dtype == FUS_DT_BF16) return FUS_D(__nv_bfloat16);
  if (dtype == FUS_DT_F16) return FUS_D(__half);
  return FUS_D(float);
#undef FUS_D
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
