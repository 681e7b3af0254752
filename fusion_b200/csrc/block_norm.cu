// The norms around a block, with its gate and residual scale, in one pass over the rows:
//   v = y / sqrt(mean(y^2) + eps) * post_w        (post_w NULL: v = y)
//   h = res + alpha * act(gate) * v
//   x = h / sqrt(mean(h^2) + eps) * pre_w         (x NULL: not computed)
// Bound: HBM, 2 reads and 2 writes of an element (a full gate adds a read). A row belongs to one
// CTA and stays in registers through both sums of squares, so nothing is read twice; fp32
// throughout, h and x are each rounded once, x from the unrounded h.
#include "dtype.cuh"
#include "host_util.h"

namespace fus {
namespace {

struct NormArgs {
  const void *y, *res, *post_w, *pre_w, *gate;
  void *h, *x;
  long ldy, ldr, ldh, ldx, ldg;
  int N;
  int gate_kind;  // 0 none, 1 one for a token, 2 one for a channel, 3 one for an element
  int act;
  float alpha, eps;
};

FUS_DEVICE float gate_act(float g, int act) {
  if (act == FUS_GATE_SIGMOID) return __fdividef(1.0f, 1.0f + __expf(-g));
  if (act == FUS_GATE_TANH) {
    // 1 - 2 / (1 + e^2g), and near zero, where that cancels, the series (its next term is below
    // 4e-7 of the value at 1/4)
    const float e = 1.0f - __fdividef(2.0f, 1.0f + __expf(2.0f * g));
    const float q = g * g;
    const float near = g + g * q * (-1.0f / 3 + q * (2.0f / 15 + q * (-17.0f / 315)));
    return fabsf(g) < 0.25f ? near : e;
  }
  return g;
}

// sum over the CTA; `red` holds one float for each warp and is free again after the next sum, over
// another `red`: that sum's barrier tells that every warp has read this one's
FUS_DEVICE float cta_sum(float v, float* red) {
  v = warp_sum(v);
  const int nw = blockDim.x >> 5;
  if (nw == 1) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (int)(threadIdx.x & 31) < nw ? red[threadIdx.x & 31] : 0.f;
  return warp_sum(v);
}

template <typename T, int V>
FUS_DEVICE void unpack_v(const uint4& u, float* f) {
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = to_f(e[j]);
}
template <typename T, int V>
FUS_DEVICE uint4 pack_v(const float* f) {
  uint4 u;
  T* e = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int j = 0; j < V; ++j) e[j] = from_f<T>(f[j]);
  return u;
}

FUS_DEVICE uint4 operator&(const uint4& a, const uint4& b) {
  return make_uint4(a.x & b.x, a.y & b.y, a.z & b.z, a.w & b.w);
}

// V elements (16 bytes) from p + i for i in [i0, i0 + V) within [0, N); whole: one load
template <typename T, int V>
FUS_DEVICE void load_v(const T* p, int i0, int N, bool whole, float* f) {
  if (whole) {
    unpack_v<T, V>(ldg_stream(p + i0), f);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = i0 + j >= 0 && i0 + j < N ? to_f(p[i0 + j]) : 0.f;
  }
}
// V elements that start `skip` elements (1 .. V - 1) into the line a, and go on in the line b
template <typename T, int V>
FUS_DEVICE uint4 shift_lines(const uint4& a, const uint4& b, int skip) {
  uint32_t r[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  const int bytes = skip * (int)sizeof(T);
  if (bytes & 8) {
#pragma unroll
    for (int j = 0; j < 6; ++j) r[j] = r[j + 2];
  }
  if (bytes & 4) {
#pragma unroll
    for (int j = 0; j < 5; ++j) r[j] = r[j + 1];
  }
  if (bytes & 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = __funnelshift_r(r[j], r[j + 1], 16);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// The same for the weights, which every row reads (kept in L1). They start on 16 bytes but
// the row does not: element i0 is `off` short of a 16-byte line, so two lines are read and
// shifted together.
template <typename T, int V>
FUS_DEVICE void load_w(const T* p, int i0, int N, bool whole, int off, float* f) {
  if (whole && off == 0) {
    unpack_v<T, V>(__ldg(reinterpret_cast<const uint4*>(p + i0)), f);
  } else if (whole && i0 + off + V <= N) {
    const uint4* line = reinterpret_cast<const uint4*>(p + i0 + off - V);
    unpack_v<T, V>(shift_lines<T, V>(__ldg(line), __ldg(line + 1), V - off), f);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = i0 + j >= 0 && i0 + j < N ? to_f(p[i0 + j]) : 0.f;
  }
}
// The 16-byte line at p, of which elements [lo, hi) belong to the row (lo == 0 or hi == V): at
// most three stores. One warp has an end of the row and its CTA's next barrier waits for it.
template <typename T, int V>
FUS_DEVICE void store_end(T* p, int lo, int hi, const uint4& u) {
  if (sizeof(T) == 4) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j >= lo && j < hi) reinterpret_cast<uint32_t*>(p)[j] = w[j];
    return;
  }
  uint16_t* q = reinterpret_cast<uint16_t*>(p);
  if (lo > 0) {  // half, word, two words
    const uint32_t w = lo & 4 ? (lo & 2 ? u.w : u.z) : (lo & 2 ? u.y : u.x);
    if (lo & 1) q[lo] = (uint16_t)(w >> 16);
    const int up = lo + (lo & 1);
    if ((up & 3) == 2) *reinterpret_cast<uint32_t*>(q + up) = up == 2 ? u.y : u.w;
    if (up <= 4) *reinterpret_cast<uint2*>(q + 4) = make_uint2(u.z, u.w);
  } else {  // two words, word, half
    if (hi & 4) *reinterpret_cast<uint2*>(q) = make_uint2(u.x, u.y);
    if (hi & 2) *reinterpret_cast<uint32_t*>(q + (hi & 4)) = hi & 4 ? u.z : u.x;
    const uint32_t w = hi & 4 ? (hi & 2 ? u.w : u.z) : (hi & 2 ? u.y : u.x);
    if (hi & 1) q[hi - 1] = (uint16_t)w;
  }
}

// lines: p + i0 starts on 16 bytes
template <typename T, int V>
FUS_DEVICE void store_v(T* p, int i0, int N, bool whole, bool lines, const float* f) {
  if (whole) {
    *reinterpret_cast<uint4*>(p + i0) = pack_v<T, V>(f);
  } else if (lines && (i0 >= 0 || i0 + V <= N)) {
    store_end<T, V>(p + i0, i0 < 0 ? -i0 : 0, N - i0 < V ? N - i0 : V, pack_v<T, V>(f));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (i0 + j >= 0 && i0 + j < N) p[i0 + j] = from_f<T>(f[j]);
  }
}

// One CTA for a row, VPT 16-byte vectors for a thread. MODE 0: every row of every tensor starts
// on 16 bytes, the weights too. 1: the weights do, rows start anywhere, but alike in all row tensors
// (odd widths): vectors follow the 16-byte lines of memory, the ones at the ends go by element. 2: by
// element, where rows do not start alike or one weight is not on 16 bytes (bf16, a weight moved by
// one element: 8192 x 6144 69 -> 254 us, 777 x 5003 11 -> 24, 64 x 6144 3.9 -> 6.3).
template <typename T, int VPT, int MODE>
__global__ void __launch_bounds__(1024) norm_gate_residual_kernel(const NormArgs a) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float red[2][32];
  const long t = blockIdx.x;
  const T* y = reinterpret_cast<const T*>(a.y) + t * a.ldy;
  const T* res = reinterpret_cast<const T*>(a.res) + t * a.ldr;
  const int N = a.N;
  const int off = MODE == 1 ? (int)((reinterpret_cast<uintptr_t>(y) & 15) / sizeof(T)) : 0;
  auto start = [&](int v) { return ((int)threadIdx.x + v * (int)blockDim.x) * V - off; };
  auto whole = [&](int i) { return MODE != 2 && i >= 0 && i + V <= N; };
  float f[VPT][V], r[VPT][V];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int i = start(v);
    if (i < N) {
      load_v<T, V>(y, i, N, whole(i), f[v]);
      load_v<T, V>(res, i, N, whole(i), r[v]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) f[v][j] = r[v][j] = 0.f;
    }
  }
  float scale = a.alpha;
  if (a.post_w) {
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int j = 0; j < V; ++j) ss += f[v][j] * f[v][j];
    ss = cta_sum(ss, red[0]);
    scale *= 1.0f / sqrtf(ss / (float)N + a.eps);
  }
  if (a.gate_kind == 1) scale *= gate_act(to_f(reinterpret_cast<const T*>(a.gate)[t * a.ldg]), a.act);
  T* h = reinterpret_cast<T*>(a.h) + t * a.ldh;
  float sh = 0.f;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int i = start(v);
    if (i >= N) continue;
    if (a.post_w) {
      float w[V];
      load_w<T, V>(reinterpret_cast<const T*>(a.post_w), i, N, whole(i), off, w);
#pragma unroll
      for (int j = 0; j < V; ++j) f[v][j] *= w[j];
    }
    if (a.gate_kind >= 2) {
      float g[V];
      if (a.gate_kind == 2)
        load_w<T, V>(reinterpret_cast<const T*>(a.gate), i, N, whole(i), off, g);
      else
        load_v<T, V>(reinterpret_cast<const T*>(a.gate) + t * a.ldg, i, N, whole(i), g);
#pragma unroll
      for (int j = 0; j < V; ++j) f[v][j] *= gate_act(g[j], a.act);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      f[v][j] = r[v][j] + scale * f[v][j];
      sh += f[v][j] * f[v][j];
    }
    store_v<T, V>(h, i, N, whole(i), MODE == 1, f[v]);
  }
  if (!a.x) return;
  sh = cta_sum(sh, red[1]);
  const float rstd = 1.0f / sqrtf(sh / (float)N + a.eps);
  T* x = reinterpret_cast<T*>(a.x) + t * a.ldx;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int i = start(v);
    if (i >= N) continue;
    float w[V];
    load_w<T, V>(reinterpret_cast<const T*>(a.pre_w), i, N, whole(i), off, w);
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] *= f[v][j] * rstd;
    store_v<T, V>(x, i, N, whole(i), MODE == 1, w);
  }
}

// Many rows: persistent CTAs, each with a ring of rows that bulk copies fill ahead of the
// arithmetic, so that loads never wait for a row's two sums and barriers. The weights (and a
// channel gate) stay in registers over all rows. A row is up to three 16-byte lines for a thread;
// narrow rows get small CTAs, more of them on an SM, so that more rows are under way at once
// (a row's chain of barriers takes about a microsecond whatever its width).
// SHIFT: rows start anywhere, but alike in all row tensors (odd widths). The lines that hold a row
// are copied and its vectors are those lines; as the grid is a multiple of 8, all rows of a CTA
// start alike and the weights are shifted once. What lines hold beside the row is its
// neighbours', never used; the first row's first line and the last row's last are not copied
// where they reach past the tensor: those few elements are loaded one by one.
// Rows that use it: four for an SM of 192 lines or more; narrower ones, to 64 lines, once there are
// 14 for an SM (fp16, ring against not: 2443 x 521 8.7 and 11.9 us, 8192 x 1021 26.6 and 48.6;
// but 1200 x 1504 6.5 and 5.1, 8192 x 256 9.0 and 7.2).
constexpr int kRingRows = 4 * 148, kRingLines = 192;
constexpr int kNarrowRows = 14 * 148, kNarrowLines = 64;
constexpr int kRingThreads = 256;  // at most

template <typename T, bool FULL, bool SHIFT>
__global__ void __launch_bounds__(kRingThreads, 2)
    norm_gate_residual_ring_kernel(const NormArgs a, int rows, int stages, int* status) {
  constexpr int V = 16 / sizeof(T), VPT = 3;
  __shared__ float red[2][32];
  __shared__ uint64_t bars[8];
  __shared__ volatile int abort_flag;
  __shared__ __align__(16) uint4 inside[2];  // SHIFT: ones where the row's first, last line hold it
  extern __shared__ __align__(16) uint8_t ring[];  // stages x (y | res | gate)
  const int N = a.N, nt = blockDim.x;
  const int lines = (N + V - 1) / V + (SHIFT ? 1 : 0);  // at most, of a row
  const uint32_t row_bytes = (uint32_t)lines * 16;
  const uint32_t stage_bytes = row_bytes * (FULL ? 3 : 2);
  const uint32_t bar = smem_u32(bars);
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(bar + 8 * s, 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  // elements of a row's first line before the row, the same for all of this CTA's rows
  const int off = SHIFT ? (int)((reinterpret_cast<uintptr_t>(reinterpret_cast<const T*>(a.y) +
                                                             blockIdx.x * a.ldy) & 15) / sizeof(T))
                        : 0;
  const int row_lines = (N + off + V - 1) / V;
  if (SHIFT && threadIdx.x < 32) {  // each byte
    const int end = threadIdx.x >> 4, j = (threadIdx.x & 15) / (int)sizeof(T);
    const bool in = end == 0 ? j >= off : j < N + off - (row_lines - 1) * V;
    reinterpret_cast<uint8_t*>(inside)[threadIdx.x] = in ? 0xff : 0;
  }
  __syncthreads();
  auto load_row = [&](long t, int s) {
    const uint64_t pol = policy_evict_first();
    const int l0 = SHIFT && t == 0 && off > 0;
    const int l1 = SHIFT && t == rows - 1 ? (N + off) / V : row_lines;
    const uint32_t bytes = (uint32_t)(l1 - l0) * 16;
    const uint32_t dst = smem_u32(ring) + s * stage_bytes + l0 * 16;
    const long from = (long)l0 * V - off;
    mbar_arrive_expect_tx(bar + 8 * s, bytes * (FULL ? 3 : 2));
    bulk_load(dst, reinterpret_cast<const T*>(a.y) + t * a.ldy + from, bytes, bar + 8 * s, pol);
    bulk_load(dst + row_bytes, reinterpret_cast<const T*>(a.res) + t * a.ldr + from, bytes,
              bar + 8 * s, pol);
    if (FULL)
      bulk_load(dst + 2 * row_bytes, reinterpret_cast<const T*>(a.gate) + t * a.ldg + from, bytes,
                bar + 8 * s, pol);
  };
  if (threadIdx.x == 0)
    for (int s = 0; s < stages; ++s) {
      const long t = blockIdx.x + (long)s * gridDim.x;
      if (t < rows) load_row(t, s);
    }
  // first element of this thread's line v, negative before the row
  auto first = [&](int v) { return ((int)threadIdx.x + v * nt) * V - off; };
  auto whole = [&](int i) { return !SHIFT || (i >= 0 && i + V <= N); };
  // not kept in L2 for long (8192 x 6144 bf16: 76 -> 69 us)
  auto put = [&](T* p, int i, const float* f) {
    const uint4 u = pack_v<T, V>(f);
    if (whole(i))
      __stcs(reinterpret_cast<uint4*>(p + i), u);
    else
      store_end<T, V>(p + i, i < 0 ? -i : 0, N - i < V ? N - i : V, u);
  };
  // post_w times a channel gate, and pre_w, of this thread's elements
  float post[VPT][V];
  uint4 pre[VPT];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int i = first(v);
    auto take = [&](const void* p) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (!p || i >= N) return u;
      const T* w = reinterpret_cast<const T*>(p);
      if (!SHIFT) return __ldg(reinterpret_cast<const uint4*>(w + i));
      T* e = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (i + j >= 0 && i + j < N) e[j] = w[i + j];
      return u;
    };
    pre[v] = take(a.pre_w);
    unpack_v<T, V>(take(a.post_w), post[v]);
    float g[V];
    if (a.gate_kind == 2) unpack_v<T, V>(take(a.gate), g);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (!a.post_w) post[v][j] = 1.f;
      if (a.gate_kind == 2) post[v][j] *= gate_act(g[j], a.act);
    }
  }
  int n = 0;
  for (long t = blockIdx.x; t < rows; t += gridDim.x, ++n) {
    const int s = n % stages;
    float scale = a.alpha;
    if (a.gate_kind == 1)
      scale *= gate_act(to_f(reinterpret_cast<const T*>(a.gate)[t * a.ldg]), a.act);
    if (!mbar_wait_bounded(bar + 8 * s, (n / stages) & 1, &abort_flag, status)) break;
    const uint4* sy = reinterpret_cast<const uint4*>(ring + s * stage_bytes);
    const uint4* sr = sy + lines;
    const uint4* sg = sr + lines;
    float f[VPT][V];
    uint4 r[VPT], g[VPT];
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int i = first(v);
      uint4 u = make_uint4(0, 0, 0, 0);
      r[v] = g[v] = u;
      if (i < N) {
        const int l = threadIdx.x + v * nt;
        u = sy[l];
        r[v] = sr[l];
        if (FULL) g[v] = sg[l];
        if (SHIFT && !whole(i)) {
          // an end of the row: what was not copied (see above), and zeros outside the row
          if ((i < 0 && t == 0) || (i + V > N && t == rows - 1)) {
            T* e = reinterpret_cast<T*>(&u);
            T* er = reinterpret_cast<T*>(&r[v]);
            T* eg = reinterpret_cast<T*>(&g[v]);
#pragma unroll
            for (int j = 0; j < V; ++j)
              if (i + j >= 0 && i + j < N) {
                e[j] = (reinterpret_cast<const T*>(a.y) + t * a.ldy)[i + j];
                er[j] = (reinterpret_cast<const T*>(a.res) + t * a.ldr)[i + j];
                if (FULL) eg[j] = (reinterpret_cast<const T*>(a.gate) + t * a.ldg)[i + j];
              }
          }
          const uint4 in = inside[i >= 0];
          u = u & in;
          r[v] = r[v] & in;
          if (FULL) g[v] = g[v] & in;
        }
      }
      unpack_v<T, V>(u, f[v]);
#pragma unroll
      for (int j = 0; j < V; ++j) ss += f[v][j] * f[v][j];
    }
    // the row's second sum, or without one the next row's first, takes the other array
    ss = cta_sum(ss, red[a.x ? 0 : n & 1]);
    __syncwarp();  // with the sum's barrier: the whole CTA has read the stage
    if (threadIdx.x == 0) {
      const long next = t + (long)stages * gridDim.x;
      if (next < rows) load_row(next, s);
    }
    if (a.post_w) scale *= 1.0f / sqrtf(ss / (float)N + a.eps);
    float sh = 0.f;
    T* h = reinterpret_cast<T*>(a.h) + t * a.ldh;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int i = first(v);
      float w[V];
#pragma unroll
      for (int j = 0; j < V; ++j) f[v][j] *= post[v][j];
      if (FULL) {
        unpack_v<T, V>(g[v], w);
#pragma unroll
        for (int j = 0; j < V; ++j) f[v][j] *= gate_act(w[j], a.act);
      }
      unpack_v<T, V>(r[v], w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        f[v][j] = w[j] + scale * f[v][j];
        sh += f[v][j] * f[v][j];
      }
      if (i < N) put(h, i, f[v]);
    }
    if (!a.x) continue;
    sh = cta_sum(sh, red[1]);
    const float rstd = 1.0f / sqrtf(sh / (float)N + a.eps);
    T* x = reinterpret_cast<T*>(a.x) + t * a.ldx;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int i = first(v);
      float w[V];
      unpack_v<T, V>(pre[v], w);
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] *= f[v][j] * rstd;
      if (i < N) put(x, i, w);
    }
  }
}

template <typename T, bool FULL, bool SHIFT>
int launch_ring(const NormArgs& a, int rows, int threads, int stages, int bytes, cudaStream_t st,
                int* status) {
  auto fn = norm_gate_residual_ring_kernel<T, FULL, SHIFT>;
  // the limit is set once, to what the largest CTA may have
  if (int rc = ensure_smem_attr((const void*)fn, 110 * 1024, "norm_gate_residual")) return rc;
  // 512 threads on an SM; a multiple of 8 (see the kernel) unless every row has its own CTA
  const int grid = num_sms() * (2 * kRingThreads / threads) / 8 * 8;
  fn<<<grid < rows ? grid : rows, threads, bytes, st>>>(a, rows, stages, status);
  return check_launch("norm_gate_residual");
}

template <typename T>
int launch_ring_of(const NormArgs& a, int rows, int threads, int stages, int bytes, bool shift,
                   cudaStream_t st, int* status) {
  if (a.gate_kind == 3)
    return shift ? launch_ring<T, true, true>(a, rows, threads, stages, bytes, st, status)
                 : launch_ring<T, true, false>(a, rows, threads, stages, bytes, st, status);
  return shift ? launch_ring<T, false, true>(a, rows, threads, stages, bytes, st, status)
               : launch_ring<T, false, false>(a, rows, threads, stages, bytes, st, status);
}

template <typename T, int VPT>
void launch_mode(const NormArgs& a, int T_, int threads, int mode, cudaStream_t st) {
  if (mode == 0)
    norm_gate_residual_kernel<T, VPT, 0><<<T_, threads, 0, st>>>(a);
  else if (mode == 1)
    norm_gate_residual_kernel<T, VPT, 1><<<T_, threads, 0, st>>>(a);
  else
    norm_gate_residual_kernel<T, VPT, 2><<<T_, threads, 0, st>>>(a);
}

template <typename T>
int launch_norm(const NormArgs& a, int rows, cudaStream_t st, int* status) {
  constexpr int V = 16 / sizeof(T);
  // alignment of the row tensors: mode 0 wants all on 16 bytes, mode 1 alike (the weights always)
  const void* rowp[5] = {a.y, a.res, a.h, a.x, a.gate_kind == 3 ? a.gate : nullptr};
  const long rowl[5] = {a.ldy, a.ldr, a.ldh, a.ldx, a.ldg};
  bool on16 = true, alike = true;
  for (int i = 0; i < 5; ++i) {
    if (!rowp[i]) continue;
    on16 = on16 && aligned16(rowp[i]) && rowl[i] % V == 0;
    alike = alike && ((uintptr_t)rowp[i] & 15) == ((uintptr_t)a.y & 15) &&
            (rowl[i] - a.ldy) % V == 0;
  }
  const void* wp[3] = {a.post_w, a.pre_w, a.gate_kind == 2 ? a.gate : nullptr};
  bool w16 = true;
  for (const void* p : wp) w16 = w16 && (!p || aligned16(p));
  const int mode = !w16 ? 2 : on16 ? 0 : alike ? 1 : 2;
  const int nv = (a.N + V - 1) / V + (mode == 1 ? 1 : 0);
  // the ring: some rows for each CTA, rows of some lines, two stages at least
  const bool shift = mode != 0 || a.N % V != 0;
  const int lines = (a.N + V - 1) / V + (shift ? 1 : 0);
  if (mode < 2 && lines <= 3 * kRingThreads &&
      ((rows >= kRingRows && lines >= kRingLines) || (rows >= kNarrowRows && lines >= kNarrowLines))) {
    const int threads = (lines + 95) / 96 * 32;
    const int stage = lines * 16 * (a.gate_kind == 3 ? 3 : 2);
    // all of an SM's CTAs resident at once: each has 1 KB reserved and some 400 bytes static beside
    int stages = (222 * 1024 / (2 * kRingThreads / threads) - 1536) / stage;
    if (stages > 8) stages = 8;
    if (stages >= 2) return launch_ring_of<T>(a, rows, threads, stages, stages * stage, shift, st, status);
  }
  // few rows: as many threads as there are vectors (latency); many: two vectors for each
  int vpt = rows <= 2 * 148 ? 1 : 2;
  while (vpt > 1 && nv < 32 * vpt) vpt >>= 1;
  while ((nv + vpt - 1) / vpt > 1024) vpt <<= 1;
  const int threads = ((nv + vpt - 1) / vpt + 31) / 32 * 32;
  switch (vpt) {
    case 1: launch_mode<T, 1>(a, rows, threads, mode, st); break;
    case 2: launch_mode<T, 2>(a, rows, threads, mode, st); break;
    case 4: launch_mode<T, 4>(a, rows, threads, mode, st); break;
    default: return set_error(FUS_E_UNSUPPORTED, "norm_gate_residual: N=%d too wide", a.N);
  }
  return check_launch("norm_gate_residual");
}

}  // namespace
}  // namespace fus

using namespace fus;

extern "C" int fus_norm_gate_residual(const void* y, long ldy, const void* res, long ldr,
                                      const void* post_w, const void* gate, long ldg,
                                      int gate_kind, int gate_act, float alpha, void* h, long ldh,
                                      const void* pre_w, void* x, long ldx, int T, int N,
                                      int dtype, float eps, void* stream, int* status) {
  if (T < 0 || N < 1) return set_error(FUS_E_INVALID, "norm_gate_residual: bad sizes");
  if (!dtype_known(dtype)) return set_error(FUS_E_INVALID, "norm_gate_residual: dtype %d", dtype);
  if (gate_kind < FUS_GATE_NONE || gate_kind > FUS_GATE_FULL || gate_act < FUS_GATE_LINEAR ||
      gate_act > FUS_GATE_TANH)
    return set_error(FUS_E_INVALID, "norm_gate_residual: unknown gate");
  if (T == 0) return FUS_OK;
  if (!y || !res || !h || (gate_kind != FUS_GATE_NONE && !gate))
    return set_error(FUS_E_INVALID, "norm_gate_residual: null pointer");
  if ((x != nullptr) != (pre_w != nullptr))
    return set_error(FUS_E_INVALID, "norm_gate_residual: x and pre_w go together");
  if (T > 1 && (ldy < N || ldr < N || ldh < N || (x && ldx < N) ||
                (gate_kind == FUS_GATE_FULL && ldg < N) || (gate_kind == FUS_GATE_TOKEN && ldg < 0)))
    return set_error(FUS_E_INVALID, "norm_gate_residual: rows overlap");
  const void* all[7] = {y, res, post_w, gate, h, pre_w, x};
  for (const void* p : all)
    if ((uintptr_t)p % dtype_size(dtype))
      return set_error(FUS_E_INVALID, "norm_gate_residual: misaligned pointer");
  NormArgs a{y, res, post_w, pre_w, gate_kind ? gate : nullptr, h, x, ldy, ldr, ldh, ldx, ldg,
             N, gate_kind, gate_act, alpha, eps};
  cudaStream_t st = as_stream(stream);
  if (dtype == FUS_DT_BF16) return launch_norm<__nv_bfloat16>(a, T, st, status);
  if (dtype == FUS_DT_F16) return launch_norm<__half>(a, T, st, status);
  return launch_norm<float>(a, T, st, status);
}
