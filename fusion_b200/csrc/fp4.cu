// Quantisation to and from microscaled 4-bit floating point (formats and scale layout:
// fp4.cuh), and the packing of a checkpoint's row-major scales into scale tiles.
//
// Mathematics, for a block with largest magnitude a:
//   MX  s = 2^(floor(log2 a) - 2) (0 for a = 0), clamped to [2^-127, 2^127]
//   NV  s = e4m3(a / (6 g)), to the nearest, ties to even, at most 448
//   q = e2m1(x / s) or e2m1(x / (s g)), to the nearest, ties to even, at most 6
// Every code is the one of exact arithmetic. MX only scales by powers of two, which fp32 does
// exactly. NV divides: fp32 leaves a relative error below 2^-21, so the quotient is rounded
// twice, a little smaller and a little larger (1 -+ 2^-21); where the two codes differ, the
// value is compared with the border between them times s g, a product and its rounding error.
// That is not rare: a factor taken from a bf16 maximum makes exact ties of bf16 values (half
// of the warps of a 8192 x 6144 tensor meet one), so it must be cheap (the comparison in
// fp64 cost 19 of 57 us there).
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

// 16 consecutive elements; vec: p is 32-byte aligned
template <typename T>
FUS_DEVICE void load16(const T* p, bool vec, uint32_t* r) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      ld32(reinterpret_cast<const char*>(p) + 32 * i, r + 8 * i);
  } else {
    T* e = reinterpret_cast<T*>(r);
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = p[i];
  }
}

// the largest magnitude's bits (fp32). Magnitudes compare as integers: an infinity or NaN comes
// out on top.
template <typename T>
FUS_DEVICE uint32_t top16(const uint32_t* r) {
  uint32_t top = 0;
  if constexpr (sizeof(T) == 2) {  // two 16-bit magnitudes at a time
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __vmaxu2(top, r[i] & 0x7fff7fffu);
    const uint16_t m = (uint16_t)max(top & 0xffffu, top >> 16);
    return __float_as_uint(to_f(*reinterpret_cast<const T*>(&m)));
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, r[i] & 0x7fffffffu);
    return top;
  }
}

// element j, by selection (no indexed registers)
template <typename T>
FUS_DEVICE float pick16(const uint32_t* r, int j) {
  constexpr int W = 8 * sizeof(T) / 2;  // words
  const int w = sizeof(T) == 2 ? j >> 1 : j;
  uint32_t v[W];
#pragma unroll
  for (int i = 0; i < W; ++i) v[i] = r[i];
#pragma unroll
  for (int n = W / 2, bit = W / 2; n > 0; n >>= 1, bit >>= 1)
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = w & bit ? v[i + n] : v[i];
  if (sizeof(T) == 2) v[0] >>= 16 * (j & 1);
  return to_f(*reinterpret_cast<const T*>(v));
}

// eight e2m1 codes of f * m, the first in the low four bits; two products an instruction
template <typename T>
FUS_DEVICE uint32_t cvt8(const uint32_t* r, float m) {
  const T* f = reinterpret_cast<const T*>(r);
  uint32_t v;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t.reg .b64 s, p;\n\t.reg .f32 lo, hi;\n\t"
      "mov.b64 s, {%9, %9};\n\t"
      "mov.b64 p, {%1, %2};\n\tmul.rn.f32x2 p, p, s;\n\tmov.b64 {lo, hi}, p;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, hi, lo;\n\t"
      "mov.b64 p, {%3, %4};\n\tmul.rn.f32x2 p, p, s;\n\tmov.b64 {lo, hi}, p;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, hi, lo;\n\t"
      "mov.b64 p, {%5, %6};\n\tmul.rn.f32x2 p, p, s;\n\tmov.b64 {lo, hi}, p;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, hi, lo;\n\t"
      "mov.b64 p, {%7, %8};\n\tmul.rn.f32x2 p, p, s;\n\tmov.b64 {lo, hi}, p;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, hi, lo;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(v)
      : "f"(to_f(f[0])), "f"(to_f(f[1])), "f"(to_f(f[2])), "f"(to_f(f[3])), "f"(to_f(f[4])),
        "f"(to_f(f[5])), "f"(to_f(f[6])), "f"(to_f(f[7])), "f"(m));
  return v;
}

// a > u g, or a = u g and `tie`: exact in fp32 where a is within 2^-20 of u g, u has a few
// bits and u g is far from fp32's ends (the product's rounding error is one more fp32 number,
// the difference is exact)
FUS_DEVICE bool above(float a, float u, float g, bool tie) {
  const float prod = u * g, err = fmaf(u, g, -prod), d = a - prod;
  return d > err || (d == err && tie);
}

FUS_DEVICE float rcp_approx(float v) {  // within 2^-23 of 1 / v
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// e4m3 byte nearest to a / (6 g), ties to even, at most 448; g is far from fp32's ends, inv6g =
// 1 / (6 g). The quotient need not be: all that is past 448 is held there, infinity too, before it
// is moved by its error (infinity less infinity would be a NaN).
FUS_DEVICE uint32_t nv_scale(float a, float g, float inv6g) {
  const float t = fminf(a * inv6g, 512.0f);
  constexpr float kEps = 1.0f / (1 << 21);
  const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(t - t * kEps, t + t * kEps),
                                                __NV_SATFINITE, __NV_E4M3);
  const uint32_t b0 = two & 0xff, b1 = two >> 8;
  if (b0 == b1) return b0;
  const float u = 3.0f * (fp4_scale_value<FUS_FP4_NV>(b0) + fp4_scale_value<FUS_FP4_NV>(b1));
  return above(a, u, g, b0 & 1) ? b1 : b0;
}
// Byte and sixteen codes for a factor near fp32's ends (or not positive: zeros), in fp64: all
// products below are exact there.
template <typename T>
FUS_DEVICE uint64_t nv_exact(const uint32_t* r, float a, float g, uint32_t* byte) {
  uint32_t b = 126;  // the grid is monotone in the byte: step down to the nearest
  while (b > 0) {
    const double m = 3.0 * (double)g * ((double)fp4_scale_value<FUS_FP4_NV>(b) +
                                        (double)fp4_scale_value<FUS_FP4_NV>(b - 1));
    if ((double)a > m || ((double)a == m && (b & 1) == 0)) break;
    --b;
  }
  *byte = b;
  const double p = (double)fp4_scale_value<FUS_FP4_NV>(b) * (double)g;
  uint64_t codes = 0;
#pragma unroll 1
  for (int j = 0; j < 16 && p > 0.0; ++j) {
    const float f = pick16<T>(r, j);
    const double v = fabs((double)f);
    uint64_t c = (v > 0.25 * p) + (v >= 0.75 * p) + (v > 1.25 * p) + (v >= 1.75 * p) +
                 (v > 2.5 * p) + (v >= 3.5 * p) + (v > 5.0 * p);
    c |= (uint64_t)(__float_as_uint(f) >> 31) << 3;
    codes |= c << (4 * j);
  }
  return codes;
}

// sixteen codes of x / (s g): `lo` and `hi` are the codes a little below and above; where they
// differ (by one) the border between them decides. A thread has one such element, rarely two:
// they are visited one by one, not in sixteen tests.
template <typename T>
FUS_DEVICE uint64_t resolve16(uint64_t lo, uint64_t hi, const uint32_t* r, float s, float g) {
  uint64_t differ = lo ^ hi;
  while (differ) {
    const int sh = (__ffsll((long long)differ) - 1) & ~3;
    const uint32_t c = (uint32_t)(lo >> sh) & 7u;
    const float border = c < 4 ? 0.25f + 0.5f * (float)c : c == 4 ? 2.5f : c == 5 ? 3.5f : 5.0f;
    const uint64_t mask = (uint64_t)15 << sh;
    if (above(fabsf(pick16<T>(r, sh >> 2)), border * s, g, c & 1)) lo = (lo & ~mask) | (hi & mask);
    differ &= ~mask;
  }
  return lo;
}

// place of every (token, slot) pair in the dispatch order: pos[id] = p where ids[p] = id. Pairs
// that are not placed keep junk; the reader checks ids[pos[id]] = id.
__global__ void fp4_invert_kernel(const int* __restrict__ ids, const int* __restrict__ ntp, int cap,
                                  int limit, int* __restrict__ pos) {
  const int used = ntp ? min(__ldg(ntp), cap) : cap;
  const int p = blockIdx.x * blockDim.x + threadIdx.x;
  if (p >= used) return;
  const int id = __ldg(ids + p);
  if (id >= 0 && id < limit) pos[id] = p;
}

// One thread quantises 16 elements of `iters` rows; blockDim (UX, 256 / UX), UX a power of two
// >= 16 that divides the row's padded K / 16, so a row's 256 elements are 16 neighbouring lanes
// and the scale bytes of a cell, in four (NV) or eight (MX) of them, leave as one 4-byte store.
// Bound: HBM (2.56 bytes an element from bf16) and, close behind, instruction issue: what
// does not depend on the row is computed once for several rows.
// SPREAD: the rows are tokens, each written to the places of its id_div (token, slot) pairs in
// the dispatch order, pos[] (checked against ids[]).
template <typename T, int FMT, bool SPREAD>
__global__ void __launch_bounds__(256)
    fp4_quantize_kernel(const T* __restrict__ x, int ldx, int x_rows, int rows, int iters,
                        const int* __restrict__ ntp, const int* __restrict__ ids, int id_div,
                        int id_limit, const int* __restrict__ pos, int K,
                        const float* __restrict__ gscale, int rows_per_g,
                        int tile_log2, uint8_t* __restrict__ q, int ldq,
                        uint8_t* __restrict__ sf, int vec, int* status) {
  pdl_allow_dependents();
  const int k = (blockIdx.y * blockDim.x + threadIdx.x) * 16;
  const int used = !SPREAD && ntp ? min(__ldg(ntp), rows) : rows;
  const int placed = SPREAD && ntp ? __ldg(ntp) : 0x7fffffff;
  const int j0 = k / fp4_block(FMT);  // this thread's scale
  const int tile = 1 << tile_log2;
  const long per_tile = (long)gridDim.y * blockDim.x / 16 * fp4_stage_scale_bytes(FMT, tile);
  constexpr int kLanes = FMT == FUS_FP4_MX ? 8 : 4;
  const int shift = 8 * ((threadIdx.x / (kLanes / 4)) & 3);
  uint8_t* cells = sf + fp4_scale_offset(tile, 0, j0 & ~3);
  x += k;
  q += k / 2;
  float g = gscale && rows_per_g == 0 ? __ldg(gscale) : 1.0f;
  float inv6g = 1.0f / (6.0f * g);
  const int p0 = blockIdx.x * blockDim.y * iters + threadIdx.y;
  constexpr int W = 8 * sizeof(T) / 2;
  constexpr int HALF = W / 2;
  // The row after the one at work is on its way (8192 x 6144 bf16: MX 24.8 -> 22.9 us, NV 36 -> 34).
  // NV from fp32 needs those registers for occupancy instead (48.4 -> 40 us).
  constexpr bool kAhead = FMT == FUS_FP4_MX || sizeof(T) == 2;
  uint32_t next[W];
  bool next_live = false;
  auto fetch = [&](int p) {
    next_live = p < used;
    int src = p;
    if (!SPREAD && next_live && ids) {
      const int id = __ldg(ids + p);
      next_live = id >= 0 && id < id_limit;  // dispatch pads keep what their rows held
      src = id_div > 1 ? id / id_div : id;
      if (next_live && src >= x_rows) {
        raise_status(status, FUS_ERR_CAPACITY);
        next_live = false;
      }
    }
    if (next_live && k < K) {
      load16(x + (long)src * ldx, vec, next);
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) next[j] = 0;
    }
  };
  if (kAhead) fetch(p0);
#pragma unroll 1
  for (int i = 0; i < iters; ++i) {
    const int p = p0 + i * blockDim.y;
    if (!kAhead) fetch(p);
    uint32_t f[W];
#pragma unroll
    for (int j = 0; j < W; ++j) f[j] = next[j];
    const bool live = next_live;
    const bool data = live && k < K;
    if (kAhead && i + 1 < iters) fetch(p + blockDim.y);
    uint32_t top = top16<T>(f);
    if (FMT == FUS_FP4_MX) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const bool bad = top >= 0x7f800000u;  // infinity or NaN in the block
    uint32_t byte = 0;
    uint2 c = make_uint2(0, 0);
    if (FMT == FUS_FP4_MX) {
      const int e = (int)(top >> 23) - 2;
      byte = e > 0 ? e : 0;
      const float inv = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte)
      c = make_uint2(cvt8<T>(f, inv), cvt8<T>(f + HALF, inv));
    } else if (data) {
      if (rows_per_g) {
        g = __ldg(gscale + p / rows_per_g);
        inv6g = 1.0f / (6.0f * g);
      }
      const float a = bad ? 0.f : __uint_as_float(top);
      if (g > 1e-30f && g < 1e30f) {
        byte = nv_scale(a, g, inv6g);
        const float s = fp4_scale_value<FUS_FP4_NV>(byte);
        // s = 0 only for magnitudes below 6 g 2^-10: their codes are zeros
        const float inv = s > 0.f ? rcp_approx(s * g) : 0.f;
        constexpr float kLo = 1.0f - 1.0f / (1 << 21), kHi = 1.0f + 1.0f / (1 << 21);
        c = make_uint2(cvt8<T>(f, inv * kLo), cvt8<T>(f + HALF, inv * kLo));
        const uint2 up = make_uint2(cvt8<T>(f, inv * kHi), cvt8<T>(f + HALF, inv * kHi));
        if ((c.x != up.x || c.y != up.y) && !bad) {
          const uint64_t r = resolve16<T>((uint64_t)c.y << 32 | c.x,
                                          (uint64_t)up.y << 32 | up.x, f, s, g);
          c = make_uint2((uint32_t)r, (uint32_t)(r >> 32));
        }
      } else {
        const uint64_t r = nv_exact<T>(f, a, g, &byte);
        c = make_uint2((uint32_t)r, (uint32_t)(r >> 32));
      }
    }
    if (bad) {
      byte = FMT == FUS_FP4_MX ? 255 : 127;
      c = make_uint2(0, 0);
    }
    // scales: NV one byte of each lane, MX one of each lane pair; zeros past K
    if (!data) byte = 0;
    uint32_t word = byte << shift;
#pragma unroll
    for (int o = kLanes / 4; o < kLanes; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
    if (!live) continue;
    auto put = [&](int d) {
      if (data) *reinterpret_cast<uint2*>(q + (long)d * ldq) = c;
      if (tile_log2 == 0) {
        if (k < K && (FMT == FUS_FP4_NV || (threadIdx.x & 1) == 0))
          sf[(long)d * (K / fp4_block(FMT)) + j0] = (uint8_t)byte;
      } else if ((threadIdx.x & (kLanes - 1)) == 0) {
        *reinterpret_cast<uint32_t*>(cells + (d >> tile_log2) * per_tile +
                                     fp4_row_offset(d & (tile - 1))) = word;
      }
    };
    if constexpr (!SPREAD) {
      put(p);
    } else {
      // the places of four pairs at a time: their loads do not wait for one another
      for (int s0 = 0; s0 < id_div; s0 += 4) {
        int d[4];
        bool is[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int id = p * id_div + s0 + u;
          is[u] = s0 + u < id_div && id < id_limit;
          d[u] = is[u] ? __ldg(pos + id) : -1;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          is[u] = is[u] && d[u] >= 0 && d[u] < x_rows && d[u] < placed &&
                  __ldg(ids + d[u]) == p * id_div + s0 + u;
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (is[u]) put(d[u]);
      }
    }
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
    fp4_dequantize_kernel(const uint8_t* __restrict__ q, int ldq, const uint8_t* __restrict__ sf,
                          int tile_log2, int rows, int iters, int K,
                          const float* __restrict__ gscale, int rows_per_g, T* __restrict__ out,
                          int ldo, int vec) {
  const int k = (blockIdx.y * blockDim.x + threadIdx.x) * 16;
  if (k >= K) return;
  const int j0 = k / fp4_block(FMT);
  const int tile = 1 << tile_log2;
  const long per_tile = (long)gridDim.y * blockDim.x / 16 * fp4_stage_scale_bytes(FMT, tile);
  const int n_scales = K / fp4_block(FMT);
  sf += tile_log2 ? fp4_scale_offset(tile, 0, j0) : j0;
  q += k / 2;
  out += k;
  float m = FMT == FUS_FP4_NV && gscale && rows_per_g == 0 ? __ldg(gscale) : 1.0f;
  const int p0 = blockIdx.x * blockDim.y * iters + threadIdx.y;
#pragma unroll 2
  for (int i = 0; i < iters; ++i) {
    const int p = p0 + i * blockDim.y;
    if (p >= rows) return;
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(q + (long)p * ldq));
    const uint32_t byte = __ldg(sf + (tile_log2 ? (p >> tile_log2) * per_tile + fp4_row_offset(p & (tile - 1))
                                                : (long)p * n_scales));
    uint32_t o[8 * sizeof(T) / 2];
    T* e = reinterpret_cast<T*>(o);
    __half2 hs;
    if (FMT == FUS_FP4_MX) {
      m = fp4_scale_value<FMT>(byte);
    } else {
      if (rows_per_g) m = __ldg(gscale + p / rows_per_g);
      const __half_raw r = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3);
      hs = __half2half2(*reinterpret_cast<const __half*>(&r));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2(
          (__nv_fp4x2_storage_t)((j < 4 ? v.x >> (8 * j) : v.y >> (8 * (j - 4))) & 0xff), __NV_E2M1);
      __half2 w = *reinterpret_cast<const __half2*>(&h);
      // value x scale is exact (NV: 6 bits, in fp16); the factor rounds once, the type once
      if (FMT == FUS_FP4_NV) w = __hmul2(w, hs);
      const float2 wf = __half22float2(w);
      e[2 * j] = from_f<T>(wf.x * m);
      e[2 * j + 1] = from_f<T>(wf.y * m);
    }
    T* dst = out + (long)p * ldo;
    if (vec) {
#pragma unroll
      for (int j = 0; j < (int)sizeof(T) / 2; ++j) st32(reinterpret_cast<char*>(dst) + 32 * j, o + 8 * j);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) dst[j] = e[j];
    }
  }
}

// row-major scales [n_experts * w_rows, K / n] -> weight scale tiles of 128 rows for each
// expert; gate_up: tile t holds gate rows [64t, 64t + 64) and their up rows, 8 and 8 in turn
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
    const int f = tl * 64 + r / 16 * 8 + r % 8;
    row = f < w_rows / 2 ? f + (r % 16 >= 8 ? w_rows / 2 : 0) : w_rows;
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

// Threads over the rows, padded to whole stages of K: (UX, 256 / UX), see the kernel. Up to
// eight rows for a thread while eight CTAs remain for each SM.
int shape_of(long rows, int K, dim3& grid, dim3& block) {
  const int per_row = (int)(fp4_stages(K) * (kFp4StageK / 16));
  int ux = 16;
  while (ux < 128 && per_row % (2 * ux) == 0) ux *= 2;
  block = dim3(ux, 256 / ux);
  const long blocks = (rows + block.y - 1) / block.y;
  int iters = 1;
  while (iters < 8 && blocks * (per_row / ux) / (2 * iters) >= 8 * 148) iters *= 2;
  grid = dim3((unsigned)((blocks + iters - 1) / iters), per_row / ux);
  return iters;
}

template <typename T>
int quantize_launch(const void* x, long ldx, int x_rows, long rows, const int* ntp, const int* ids,
                    int id_div, int id_limit, const int* pos, int K, int fmt, const float* gscale,
                    long rows_per_g, int tile, void* q, long ldq, void* sf, cudaStream_t st,
                    int* status) {
  dim3 grid, block;
  const int iters = shape_of(rows, K, grid, block);
  const int vec = (reinterpret_cast<uintptr_t>(x) % 32) == 0 && (ldx * (long)sizeof(T)) % 32 == 0;
  auto fn = pos ? (fmt == FUS_FP4_MX ? fp4_quantize_kernel<T, FUS_FP4_MX, true>
                                     : fp4_quantize_kernel<T, FUS_FP4_NV, true>)
                : (fmt == FUS_FP4_MX ? fp4_quantize_kernel<T, FUS_FP4_MX, false>
                                     : fp4_quantize_kernel<T, FUS_FP4_NV, false>);
  fn<<<grid, block, 0, st>>>(reinterpret_cast<const T*>(x), (int)ldx, x_rows, (int)rows, iters, ntp,
                             ids, id_div, id_limit, pos, K, gscale, (int)rows_per_g, log2_of(tile),
                             reinterpret_cast<uint8_t*>(q), (int)ldq,
                             reinterpret_cast<uint8_t*>(sf), vec, status);
  return check_launch("fp4_quantize");
}

template <typename T>
int dequantize_launch(const void* q, long ldq, const void* sf, int fmt, int tile, long rows, int K,
                      const float* gscale, long rows_per_g, void* out, long ldo, cudaStream_t st) {
  dim3 grid, block;
  const int iters = shape_of(rows, K, grid, block);
  const int vec = (reinterpret_cast<uintptr_t>(out) % 32) == 0 && (ldo * (long)sizeof(T)) % 32 == 0;
  auto fn = fmt == FUS_FP4_MX ? fp4_dequantize_kernel<T, FUS_FP4_MX> : fp4_dequantize_kernel<T, FUS_FP4_NV>;
  fn<<<grid, block, 0, st>>>(reinterpret_cast<const uint8_t*>(q), (int)ldq,
                             reinterpret_cast<const uint8_t*>(sf), log2_of(tile), (int)rows, iters, K,
                             gscale, (int)rows_per_g, reinterpret_cast<T*>(out), (int)ldo, vec);
  return check_launch("fp4_dequantize");
}

int check_common(const char* what, int fmt, int dtype, long rows, int K, int tile) {
  if (fmt != FUS_FP4_MX && fmt != FUS_FP4_NV)
    return set_error(FUS_E_INVALID, "%s: unknown format %d", what, fmt);
  if (!dtype_known(dtype))
    return set_error(FUS_E_INVALID, "%s: unknown dtype %d", what, dtype);
  if (rows < 0 || rows > kMaxRows) return set_error(FUS_E_INVALID, "%s: bad row count", what);
  if (K <= 0 || K % 32)
    return set_error(FUS_E_INVALID, "%s: K=%d must be a positive multiple of 32", what, K);
  if (tile != 0 && !valid_tile(tile))
    return set_error(FUS_E_INVALID, "%s: tile %d not in {0,16,32,64,128,256}", what, tile);
  return FUS_OK;
}

}  // namespace

int fp4_quantize_spread(const void* x, int dtype, long ldx, int T, int K, int fmt, const float* g,
                        const int* ids, int per_token, int limit, const int* ntp, int cap, int tile,
                        int* pos, void* q, long ldq, void* sf, void* stream, int* status) {
  cudaStream_t st = as_stream(stream);
  fp4_invert_kernel<<<(cap + 255) / 256, 256, 0, st>>>(ids, ntp, cap, limit, pos);
  if (int rc = check_launch("fp4_quantize")) return rc;
#define FUS_Q(E)                                                                                 \
  quantize_launch<E>(x, ldx, cap, T, ntp, ids, per_token, limit, pos, K, fmt, g, 0, tile, q, ldq, \
                     sf, st, status)
  if (dtype == FUS_DT_BF16) return FUS_Q(__nv_bfloat16);
  if (dtype == FUS_DT_F16) return FUS_Q(__half);
  return FUS_Q(float);
#undef FUS_Q
}

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
  if (rows == 0 || (ids && id_div > 0 && id_limit == 0)) return FUS_OK;  // no live row
  if (!x || !q || !sf) return set_error(FUS_E_INVALID, "fp4_quantize: null pointer");
  if (x_rows < 1 || ldx < K || ldx > 0x7fffffffL) return set_error(FUS_E_INVALID, "fp4_quantize: bad source rows");
  if (!ids && rows > x_rows)
    return set_error(FUS_E_INVALID, "fp4_quantize: %ld rows of %d", rows, x_rows);
  if (ids && (id_div < 1 || id_limit < 0))
    return set_error(FUS_E_INVALID, "fp4_quantize: bad id_div / id_limit");
  if (reinterpret_cast<uintptr_t>(x) % dtype_size(dtype))
    return set_error(FUS_E_INVALID, "fp4_quantize: misaligned source");
  if (ldq < K / 2 || ldq > 0x7fffffffL || ldq % 16 || !aligned16(q) || !aligned16(sf))
    return set_error(FUS_E_INVALID, "fp4_quantize: packed rows must be 16-byte aligned");
  if (rows_per_g < 0 || rows_per_g > 0x7fffffffL) return set_error(FUS_E_INVALID, "fp4_quantize: bad rows_per_g");
  if (fmt == FUS_FP4_MX && gscale)
    return set_error(FUS_E_INVALID, "fp4_quantize: FUS_FP4_MX takes no factor");
  cudaStream_t st = as_stream(stream);
#define FUS_Q(T)                                                                               \
  quantize_launch<T>(x, ldx, x_rows, rows, ntp, ids, id_div, id_limit, nullptr, K, fmt, gscale,          \
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
  if (ldq < K / 2 || ldq > 0x7fffffffL || ldq % 8 || reinterpret_cast<uintptr_t>(q) % 8)
    return set_error(FUS_E_INVALID, "fp4_dequantize: packed rows must be 8-byte aligned");
  if (ldo < K || ldo > 0x7fffffffL || reinterpret_cast<uintptr_t>(out) % dtype_size(dtype))
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
