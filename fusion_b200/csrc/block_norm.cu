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
  if (act == FUS_GATE_TANH) return tanhf(g);
  return g;
}

// sum over the CTA; `red` holds one float for each warp and is free again after the next sum
FUS_DEVICE float cta_sum(float v, float* red) {
  v = warp_sum(v);
  const int nw = blockDim.x >> 5;
  if (nw == 1) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (int)(threadIdx.x & 31) < nw ? red[threadIdx.x & 31] : 0.f;
  return warp_sum(v);
}

// V elements (16 bytes) from p + i for i in [i0, i0 + V) within [0, N); whole: one load
template <typename T, int V>
FUS_DEVICE void load_v(const T* p, int i0, int N, bool whole, float* f) {
  if (whole) {
    const uint4 u = ldg_stream(p + i0);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = to_f(e[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = i0 + j >= 0 && i0 + j < N ? to_f(p[i0 + j]) : 0.f;
  }
}
// the same for the weights, which every row reads (kept in L1)
template <typename T, int V>
FUS_DEVICE void load_w(const T* p, int i0, int N, bool whole, float* f) {
  if (whole) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p + i0));
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = to_f(e[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = i0 + j >= 0 && i0 + j < N ? to_f(p[i0 + j]) : 0.f;
  }
}
template <typename T, int V>
FUS_DEVICE void store_v(T* p, int i0, int N, bool whole, const float* f) {
  if (whole) {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int j = 0; j < V; ++j) e[j] = from_f<T>(f[j]);
    *reinterpret_cast<uint4*>(p + i0) = u;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (i0 + j >= 0 && i0 + j < N) p[i0 + j] = from_f<T>(f[j]);
  }
}

// One CTA for a row, VPT 16-byte vectors for a thread. MODE 0: every row of every tensor starts
// on 16 bytes. 1: rows start anywhere, but alike in all row tensors (odd widths): vectors
// follow the 16-byte lines of memory, the two at the ends and the weights go by element. 2: by
// element.
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
      load_w<T, V>(reinterpret_cast<const T*>(a.post_w), i, N, MODE == 0 && whole(i), w);
#pragma unroll
      for (int j = 0; j < V; ++j) f[v][j] *= w[j];
    }
    if (a.gate_kind >= 2) {
      float g[V];
      if (a.gate_kind == 2)
        load_w<T, V>(reinterpret_cast<const T*>(a.gate), i, N, MODE == 0 && whole(i), g);
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
    store_v<T, V>(h, i, N, whole(i), f[v]);
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
    load_w<T, V>(reinterpret_cast<const T*>(a.pre_w), i, N, MODE == 0 && whole(i), w);
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] *= f[v][j] * rstd;
    store_v<T, V>(x, i, N, whole(i), w);
  }
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
int launch_norm(const NormArgs& a, int rows, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  // alignment of the row tensors: mode 0 wants all on 16 bytes (weights too), mode 1 alike
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
  for (const void* p : wp) on16 = on16 && (!p || aligned16(p));
  const int mode = on16 ? 0 : alike ? 1 : 2;
  const int nv = (a.N + V - 1) / V + (mode == 1 ? 1 : 0);
  // few rows: as many threads as there are vectors (latency); many: four vectors for each
  int vpt = rows <= 2 * 148 ? 1 : 4;
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
  (void)status;
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
  if (dtype == FUS_DT_BF16) return launch_norm<__nv_bfloat16>(a, T, st);
  if (dtype == FUS_DT_F16) return launch_norm<__half>(a, T, st);
  return launch_norm<float>(a, T, st);
}
