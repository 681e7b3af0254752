// Routing to experts from logits: scores, balancing bias, groups, top-k, weights.
//   s = sigmoid(l) or softmax(l);  c = s + bias
//   groups: the topk_group groups with the largest sum of their two largest c; others are out
//   ids = top-k of c, ties to the lower id;  w = s[ids] (/ sum, if renorm) * scale
//
// One warp for a token; a lane owns up to NPL consecutive experts of one group, so a group is a
// power-of-two run of lanes. Bound: instruction issue (a token's 256 fp32 logits are 1 KB, 0.16
// ns of HBM; the warp issues some hundreds of instructions for it). The selection therefore
// avoids k rounds over all experts: the k-th largest of the 32 lane maxima bounds the k-th
// largest expert from below, so only experts at or above it (about k + 2 of 256) are
// compacted into shared memory, one to a lane, and ranked against one another.
//
// The ids are those of exact arithmetic on the logits. Without bias and groups the logits are
// ranked themselves (the score is monotone in them). Otherwise fp32 scores rank, and where two
// choices that decide something lie within their error of each other (a few tokens in a
// thousand) the warp does the row again in fp64. The same path takes rows with more than 32
// candidates (ties) or fewer than k finite choices.
//
// A logit of -infinity or NaN masks its expert; a slot for which no expert is left gets id -1
// (a hole of the dispatch layout) and weight 0.
#include "dtype.cuh"
#include "host_util.h"

namespace fus {
namespace {

struct RouteArgs {
  const void* logits;
  long ld;
  const float* bias;
  float* topw;
  int* topi;
  int T, E, topk;
  int softmax;
  int n_group, topk_group;
  int gsz;   // experts of a group
  int lpg;   // lanes of a group (a power of two)
  int npl;   // experts of a lane
  float scale;
  int renorm;
};

constexpr int kWarps = 4;
constexpr unsigned kAll = 0xffffffffu;

FUS_DEVICE float sigmoid_fast(float l) { return __fdividef(1.0f, 1.0f + __expf(-l)); }

// order-preserving unsigned key of a float
FUS_DEVICE uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
FUS_DEVICE float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// a logit as the routing sees it: NaN and -infinity mask, +infinity is the largest number
FUS_DEVICE float clean(float l) {
  if (!(l > -INFINITY)) return -INFINITY;
  return fminf(l, 3.402823466e38f);
}

// the whole row in fp64, k rounds; every lane returns after the row's outputs are written
template <typename T>
__device__ __noinline__ void route_row_exact(const RouteArgs& a, long t, int lane) {
  const T* row = reinterpret_cast<const T*>(a.logits) + t * a.ld;
  const int group = lane / a.lpg;
  const int e0 = group * a.gsz + (lane % a.lpg) * a.npl;
  const int n = group < a.n_group ? max(0, min(a.npl, (group + 1) * a.gsz - e0)) : 0;
  double top = -INFINITY;
  for (int j = 0; j < n; ++j) top = fmax(top, (double)clean(to_f(row[e0 + j])));
  for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(kAll, top, o));
  double sum = 0.0;
  if (a.softmax && top > -INFINITY) {
    for (int j = 0; j < n; ++j) sum += exp((double)clean(to_f(row[e0 + j])) - top);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
  }
  auto score = [&](int e) {
    const double l = clean(to_f(row[e]));
    return a.softmax ? exp(l - top) / sum : 1.0 / (1.0 + exp(-l));
  };
  double c[32];  // this lane's choices (local memory)
  for (int j = 0; j < n; ++j) {
    const int e = e0 + j;
    c[j] = clean(to_f(row[e])) > -INFINITY ? score(e) + (a.bias ? (double)__ldg(a.bias + e) : 0.0)
                                           : -INFINITY;
  }
  bool in = true;
  if (a.n_group > 1) {
    double a1 = -INFINITY, a2 = -INFINITY;
    for (int j = 0; j < n; ++j) {
      const double v = c[j];
      if (v > a1) {
        a2 = a1;
        a1 = v;
      } else if (v > a2) {
        a2 = v;
      }
    }
    for (int o = 1; o < a.lpg; o <<= 1) {
      const double b1 = __shfl_xor_sync(kAll, a1, o), b2 = __shfl_xor_sync(kAll, a2, o);
      const double lo = fmax(fmin(a1, b1), fmax(a2, b2));
      a1 = fmax(a1, b1);
      a2 = lo;
    }
    const double g = a2 > -INFINITY ? a1 + a2 : a1;
    int better = 0;
    for (int q = 0; q < a.n_group; ++q) {
      const double og = __shfl_sync(kAll, g, q * a.lpg);
      better += og > g || (og == g && q < group);
    }
    in = better < a.topk_group;
  }
  uint32_t taken = 0;  // bit j: this lane's expert j was chosen (npl <= 32)
  double total = 0.0;
  double mine = 0.0;   // lane s keeps slot s
  int my_id = -1;
  for (int s = 0; s < a.topk; ++s) {
    double best = -INFINITY;
    int id = 0x7fffffff;
    if (in)
      for (int j = 0; j < n; ++j) {
        if (taken >> j & 1) continue;
        const double v = c[j];
        if (v > best) {
          best = v;
          id = e0 + j;
        }
      }
    for (int o = 16; o > 0; o >>= 1) {
      const double ob = __shfl_xor_sync(kAll, best, o);
      const int oi = __shfl_xor_sync(kAll, id, o);
      if (ob > best || (ob == best && oi < id)) {
        best = ob;
        id = oi;
      }
    }
    if (!(best > -INFINITY)) break;
    if (id >= e0 && id < e0 + n) taken |= 1u << (id - e0);
    const double w = score(id);
    total += w;
    if (lane == s) {
      mine = w;
      my_id = id;
    }
  }
  if (lane < a.topk) {
    if (a.renorm) mine /= fmax(total, 1e-20);
    a.topw[t * a.topk + lane] = my_id >= 0 ? (float)(mine * (double)a.scale) : 0.f;
    a.topi[t * a.topk + lane] = my_id;
  }
}

template <typename T, int NPL>
__global__ void __launch_bounds__(kWarps * 32) route_topk_kernel(const RouteArgs a) {
  __shared__ float2 cand[kWarps][32];  // (choice, logit)
  __shared__ int cand_id[kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long t = (long)blockIdx.x * kWarps + warp;
  if (t >= a.T) return;
  const T* row = reinterpret_cast<const T*>(a.logits) + t * a.ld;
  const int group = lane / a.lpg;
  const int e0 = group * a.gsz + (lane % a.lpg) * a.npl;
  const int n = group < a.n_group ? max(0, min(a.npl, (group + 1) * a.gsz - e0)) : 0;
  float l[NPL];
  // whole aligned runs of 16 bytes where the row allows
  constexpr int V = 16 / sizeof(T);
  if (NPL % V == 0 && n == NPL && ((uintptr_t)(row + e0) & 15) == 0) {
#pragma unroll
    for (int j = 0; j < NPL / V; ++j) {
      const uint4 u = ldg_stream(row + e0 + j * V);
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < V; ++i) l[j * V + i] = clean(to_f(e[i]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < NPL; ++j) l[j] = j < n ? clean(to_f(row[e0 + j])) : -INFINITY;
  }
  float top = -INFINITY, sum = 1.f;
  if (a.softmax) {
#pragma unroll
    for (int j = 0; j < NPL; ++j) top = fmaxf(top, l[j]);
    top = value_of(__reduce_max_sync(kAll, key_of(top)));
    sum = 0.f;
#pragma unroll
    for (int j = 0; j < NPL; ++j) sum += l[j] > -INFINITY ? __expf(l[j] - top) : 0.f;
    sum = warp_sum(sum);
  }
  // choices; `tol` bounds the error of a difference of two of them (scores up to 1, fast
  // exponential and division, one addition)
  const bool plain = !a.bias && a.n_group == 1;  // the logits rank themselves
  float c[NPL];
  float tol = 0.f;
  bool again = false;
  if (plain) {
#pragma unroll
    for (int j = 0; j < NPL; ++j) c[j] = l[j];
  } else {
    const float inv = __fdividef(1.0f, sum);
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      float s = a.softmax ? __expf(l[j] - top) * inv : sigmoid_fast(l[j]);
      if (a.bias && j < n) s += __ldg(a.bias + e0 + j);
      c[j] = l[j] > -INFINITY ? s : -INFINITY;
    }
    // softmax: the sum of up to 1024 terms adds some 2^-19 of a score
    tol = a.softmax ? 8e-6f : 4e-6f;
  }
  float best = -INFINITY;
  if (a.n_group > 1) {
    float a1 = -INFINITY, a2 = -INFINITY;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      a2 = fmaxf(a2, fminf(a1, c[j]));
      a1 = fmaxf(a1, c[j]);
    }
    best = a1;
    for (int o = 1; o < a.lpg; o <<= 1) {
      const float b1 = __shfl_xor_sync(kAll, a1, o), b2 = __shfl_xor_sync(kAll, a2, o);
      a2 = fmaxf(fminf(a1, b1), fmaxf(a2, b2));
      a1 = fmaxf(a1, b1);
    }
    const float g = a2 > -INFINITY ? a1 + a2 : a1;
    const float gt = 2.f * tol * (1.f + fabsf(g));
    int better = 0;
    bool near = false;
    for (int q = 0; q < a.n_group; ++q) {
      const float og = __shfl_sync(kAll, g, q * a.lpg);
      better += og > g || (og == g && q < group);
      near |= q != group && fabsf(og - g) <= gt;
    }
    again = group < a.n_group && near && (better == a.topk_group - 1 || better == a.topk_group);
    if (better >= a.topk_group) {
      best = -INFINITY;
#pragma unroll
      for (int j = 0; j < NPL; ++j) c[j] = -INFINITY;
    }
  } else {
#pragma unroll
    for (int j = 0; j < NPL; ++j) best = fmaxf(best, c[j]);
  }
  // k-th largest lane maximum (equal maxima leave together: the bound only gets lower)
  uint32_t mine = key_of(best), bound = 0;
  for (int s = 0; s < a.topk; ++s) {
    bound = __reduce_max_sync(kAll, mine);
    if (mine == bound) mine = 0;
  }
  float limit = value_of(bound);
  again |= !(bound > key_of(-INFINITY));  // fewer than k lanes with a finite choice
  limit -= tol * (1.f + fabsf(limit));
  int count = 0;
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    const bool is = c[j] >= limit;
    const unsigned m = __ballot_sync(kAll, is);
    if (is) {
      const int at = count + __popc(m & ((1u << lane) - 1));
      if (at < 32) {
        cand[warp][at] = make_float2(c[j], l[j]);
        cand_id[warp][at] = e0 + j;
      }
    }
    count += __popc(m);
  }
  __syncwarp();
  if (__any_sync(kAll, again) || count > 32) {
    route_row_exact<T>(a, t, lane);
    return;
  }
  const float2 my = lane < count ? cand[warp][lane] : make_float2(-INFINITY, 0.f);
  const int id = lane < count ? cand_id[warp][lane] : 0x7fffffff;
  int rank = 0;
  bool near = false;
  const float my_tol = tol * (1.f + fabsf(my.x));
  for (int q = 0; q < count; ++q) {
    const float oc = cand[warp][q].x;
    const int oi = cand_id[warp][q];
    rank += oc > my.x || (oc == my.x && oi < id);
    near |= oi != id && fabsf(oc - my.x) <= my_tol;
  }
  const bool chosen = lane < count && rank < a.topk;
  if (__any_sync(kAll, chosen && near && !plain)) {
    route_row_exact<T>(a, t, lane);
    return;
  }
  float w = 0.f;
  if (chosen)
    w = a.softmax ? expf(my.y - top) / sum : 1.0f / (1.0f + expf(-my.y));
  if (a.renorm) w = w / fmaxf(warp_sum(w), 1e-20f);
  if (chosen) {
    a.topw[t * a.topk + rank] = w * a.scale;
    a.topi[t * a.topk + rank] = id;
  }
}

template <typename T>
int launch_route(const RouteArgs& a, cudaStream_t st) {
  const int grid = (a.T + kWarps - 1) / kWarps;
  if (a.npl <= 1) route_topk_kernel<T, 1><<<grid, kWarps * 32, 0, st>>>(a);
  else if (a.npl <= 2) route_topk_kernel<T, 2><<<grid, kWarps * 32, 0, st>>>(a);
  else if (a.npl <= 4) route_topk_kernel<T, 4><<<grid, kWarps * 32, 0, st>>>(a);
  else if (a.npl <= 8) route_topk_kernel<T, 8><<<grid, kWarps * 32, 0, st>>>(a);
  else if (a.npl <= 16) route_topk_kernel<T, 16><<<grid, kWarps * 32, 0, st>>>(a);
  else route_topk_kernel<T, 32><<<grid, kWarps * 32, 0, st>>>(a);
  return check_launch("route_topk");
}

}  // namespace
}  // namespace fus

using namespace fus;

extern "C" int fus_route_topk(const void* logits, int dtype, long ld, const float* bias,
                              int score, int n_group, int topk_group, float* topw, int* topi,
                              int T, int E, int topk, float scale, int renorm, void* stream,
                              int* status) {
  (void)status;
  if (T < 0 || E < 1 || topk < 1 || topk > 32 || topk > E)
    return set_error(FUS_E_INVALID, "route_topk: T=%d E=%d topk=%d (topk <= 32, <= E)", T, E, topk);
  if (!dtype_known(dtype)) return set_error(FUS_E_INVALID, "route_topk: dtype %d", dtype);
  if (score != FUS_SCORE_SIGMOID && score != FUS_SCORE_SOFTMAX)
    return set_error(FUS_E_INVALID, "route_topk: unknown score %d", score);
  if (n_group < 1 || n_group > 32 || E % n_group || topk_group < 1 || topk_group > n_group)
    return set_error(FUS_E_INVALID, "route_topk: n_group=%d (<= 32, divides E=%d) topk_group=%d",
                     n_group, E, topk_group);
  if (topk_group * (E / n_group) < topk)
    return set_error(FUS_E_INVALID, "route_topk: %d groups of %d experts hold fewer than topk=%d",
                     topk_group, E / n_group, topk);
  RouteArgs a{};
  a.gsz = E / n_group;
  a.lpg = 32;
  while (a.lpg * n_group > 32) a.lpg >>= 1;
  a.npl = (a.gsz + a.lpg - 1) / a.lpg;
  if (a.npl > 32) return set_error(FUS_E_UNSUPPORTED, "route_topk: E=%d too many experts", E);
  // 16-byte loads want whole runs: a power of two of experts for a lane
  while (a.npl & (a.npl - 1)) ++a.npl;
  if (T == 0) return FUS_OK;
  if (!logits || !topw || !topi) return set_error(FUS_E_INVALID, "route_topk: null pointer");
  if ((T > 1 && ld < E) || (uintptr_t)logits % dtype_size(dtype))
    return set_error(FUS_E_INVALID, "route_topk: bad logit rows");
  a.logits = logits;
  a.ld = ld;
  a.bias = bias;
  a.topw = topw;
  a.topi = topi;
  a.T = T;
  a.E = E;
  a.topk = topk;
  a.softmax = score == FUS_SCORE_SOFTMAX;
  a.n_group = n_group;
  a.topk_group = topk_group;
  a.scale = scale;
  a.renorm = renorm;
  cudaStream_t st = as_stream(stream);
  if (dtype == FUS_DT_BF16) return launch_route<__nv_bfloat16>(a, st);
  if (dtype == FUS_DT_F16) return launch_route<__half>(a, st);
  return launch_route<float>(a, st);
}
