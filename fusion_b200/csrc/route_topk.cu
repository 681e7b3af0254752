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
// The ids are those of 64-bit arithmetic on the logits. Without bias and groups the logits are
// ranked themselves (the score is monotone in them). Otherwise fp32 scores rank, and where two
// choices that decide something lie within their error of each other (a few tokens in a
// thousand) the warp decides again in fp64, the groups from the experts that may be their two
// largest, the experts from the candidates, one for each lane. (A warp that does so in the last
// wave is waited for: all choices of the groups, read again from memory, cost 3 of 28 us at
// 32768 x 256 with 8 groups, now 24.9.) Rows with more than 32 candidates (ties) or fewer than k
// finite choices among the lanes' largest go through k plain rounds in fp64, which is slow. Rows do
// so whatever they hold where the lanes' largest are hardly more than k: k near 32, or near the
// lanes that own experts (groups: near twice the lanes of the groups kept). 32768 tokens: 64 experts with
// k 16 17.7, 24 106, 32 252 us; 256 with k 32 324 us; 256 in 32 groups, k 8, 4 kept 26.3, 3 kept 159 us.
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
  int lpg;   // lanes of a group, 2^lpg_log2
  int lpg_log2;
  int npl;   // experts of a lane
  float scale;
  int renorm;
};

constexpr int kWarps = 4;
constexpr unsigned kAll = 0xffffffffu;

constexpr float kLog2e = 1.4426950408889634f;
FUS_DEVICE float ex2(float v) {  // 2^v, within 2 ulp
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
FUS_DEVICE float rcp(float v) {  // 1 / v, within 1 ulp
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
FUS_DEVICE float sigmoid_fast(float l) { return rcp(1.0f + ex2(-kLog2e * l)); }

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
  return fminf(fmaxf(l, -INFINITY), 3.402823466e38f);  // fmaxf drops a NaN
}

// the whole row in fp64, k rounds; every lane returns after the row's outputs are written
template <typename T>
__device__ __noinline__ void route_row_exact(const RouteArgs& a, long t, int lane) {
  const T* row = reinterpret_cast<const T*>(a.logits) + t * a.ld;
  const int group = lane >> a.lpg_log2;
  const int e0 = group * a.gsz + (lane & (a.lpg - 1)) * a.npl;
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
  const bool plain = !a.bias && a.n_group == 1;  // the logits rank themselves
  double c[32];                                  // this lane's choices (local memory)
  for (int j = 0; j < n; ++j) {
    const int e = e0 + j;
    const float l = clean(to_f(row[e]));
    c[j] = plain || !(l > -INFINITY) ? (double)l
                                     : score(e) + (a.bias ? (double)__ldg(a.bias + e) : 0.0);
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
    // the owner's score, from its logit
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

// What the fast path cannot tell apart, in fp64. These read the row again, so that the fast
// path's values never need an address.
struct ExactRow {
  double sum;  // softmax denominator
  float top;
  bool softmax;
  template <typename T>
  FUS_DEVICE ExactRow(const RouteArgs& a, const T* row, int e0, int n, float t)
      : sum(1.0), top(t), softmax(a.softmax) {
    if (!softmax) return;
    sum = 0.0;
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const float l = clean(to_f(row[e0 + j]));
      if (l > -INFINITY) sum += exp((double)l - (double)top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
  }
  FUS_DEVICE double score(float l) const {
    return softmax ? exp((double)l - (double)top) / sum : 1.0 / (1.0 + exp(-(double)l));
  }
};

// rank of this lane's group among the groups. `in`: this lane's experts that may be one of its two
// largest (bit j for expert j), `l` their logits.
template <typename T>
__device__ __noinline__ int group_rank_exact(const RouteArgs& a, const T* row, float top, int e0,
                                             int n, int group, uint32_t in, const float* l) {
  const ExactRow x(a, row, e0, n, top);
  double a1 = -INFINITY, a2 = -INFINITY;
  for (; in; in &= in - 1) {
    const int j = __ffs(in) - 1;
    if (!(l[j] > -INFINITY)) continue;
    const double v = x.score(l[j]) + (a.bias ? (double)__ldg(a.bias + e0 + j) : 0.0);
    a2 = fmax(a2, fmin(a1, v));
    a1 = fmax(a1, v);
  }
  for (int o = 1; o < a.lpg; o <<= 1) {
    const double b1 = __shfl_xor_sync(kAll, a1, o), b2 = __shfl_xor_sync(kAll, a2, o);
    a2 = fmax(fmin(a1, b1), fmax(a2, b2));
    a1 = fmax(a1, b1);
  }
  const double g = a2 > -INFINITY ? a1 + a2 : a1;
  int better = 0;
  for (int q = 0; q < a.n_group; ++q) {
    const double og = __shfl_sync(kAll, g, q * a.lpg);
    better += og > g || (og == g && q < group);
  }
  return better;
}

// rank of this lane's candidate among `count`
template <typename T>
__device__ __noinline__ int rank_exact(const RouteArgs& a, const T* row, float top, int e0, int n,
                                       float logit, int id, int count, int lane) {
  const ExactRow x(a, row, e0, n, top);
  double c = -INFINITY;
  if (lane < count) c = x.score(logit) + (a.bias ? (double)__ldg(a.bias + id) : 0.0);
  int rank = 0;
  for (int q = 0; q < count; ++q) {
    const double oc = __shfl_sync(kAll, c, q);
    const int oi = __shfl_sync(kAll, id, q);
    rank += oc > c || (oc == c && oi < id);
  }
  return rank;
}

template <typename T, int NPL, bool SOFTMAX, bool GROUPED>
__global__ void __launch_bounds__(kWarps * 32) route_topk_kernel(const __grid_constant__ RouteArgs a) {
  __shared__ __align__(16) float row_c[kWarps][NPL * 32], row_l[kWarps][NPL * 32];  // lane-major
  __shared__ unsigned long long cand[kWarps][32];  // choice (ordered) and id (lower is larger)
  __shared__ float sorted[kWarps][33];
  __shared__ int place[kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long t = (long)blockIdx.x * kWarps + warp;
  if (t >= a.T) return;
  const T* row = reinterpret_cast<const T*>(a.logits) + t * a.ld;
  const int group = GROUPED ? lane >> a.lpg_log2 : 0;
  const int e0 = GROUPED ? group * a.gsz + (lane & (a.lpg - 1)) * NPL : lane * NPL;
  const int n = group < a.n_group ? max(0, min(NPL, (group + 1) * a.gsz - e0)) : 0;
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
  float top = 0.f, inv = 1.f;
  if (SOFTMAX) {
    top = l[0];
#pragma unroll
    for (int j = 1; j < NPL; ++j) top = fmaxf(top, l[j]);
    top = value_of(__reduce_max_sync(kAll, key_of(top)));
    float sum = 0.f;
    if (top > -INFINITY) {
#pragma unroll
      for (int j = 0; j < NPL; ++j) sum += ex2(kLog2e * (l[j] - top));
    }
    inv = 1.0f / warp_sum(sum);
  }
  auto score = [&](float v) {
    return SOFTMAX ? ex2(kLog2e * (v - top)) * inv : sigmoid_fast(v);
  };
  // choices; `tol` bounds the error of a difference of two of them
  const bool plain = !a.bias && !GROUPED;  // the logits rank themselves
  float c[NPL];
  float tol = 0.f;
  if (plain) {
#pragma unroll
    for (int j = 0; j < NPL; ++j) c[j] = l[j];
  } else {
#pragma unroll
    for (int j = 0; j < NPL; ++j) c[j] = score(l[j]);
    if (a.bias) {
      if (NPL % 4 == 0 && n == NPL && ((uintptr_t)(a.bias + e0) & 15) == 0) {
#pragma unroll
        for (int j = 0; j < NPL; j += 4) {
          const float4 b = __ldg(reinterpret_cast<const float4*>(a.bias + e0 + j));
          c[j] += b.x;
          c[j + 1] += b.y;
          c[j + 2] += b.z;
          c[j + 3] += b.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < NPL; ++j)
          if (j < n) c[j] += __ldg(a.bias + e0 + j);
      }
    }
    float low = l[0];
#pragma unroll
    for (int j = 1; j < NPL; ++j) low = fminf(low, l[j]);
    if (!(low > -INFINITY)) {  // masked experts, and places past the group
#pragma unroll
      for (int j = 0; j < NPL; ++j) c[j] = l[j] > -INFINITY ? c[j] : -INFINITY;
    }
    // sigmoid: an exponential within 2 ulp and its argument's rounding (1.2e-7 of s (1 - s) |l|,
    // below 1e-7), the sum 6e-8, a reciprocal within 1.2e-7; the addition 6e-8 of the choice;
    // all twice. softmax: the sum of up to 1024 terms adds some 2^-19 of a score.
    tol = SOFTMAX ? 8e-6f : 9e-7f;
  }
  float best, second = -INFINITY;  // of this lane (second: GROUPED only)
  if (GROUPED) {
    float a1 = c[0], a2 = -INFINITY;
#pragma unroll
    for (int j = 1; j < NPL; ++j) {
      a2 = fmaxf(a2, fminf(a1, c[j]));
      a1 = fmaxf(a1, c[j]);
    }
    best = a1;
    second = a2;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      if (o >= a.lpg) break;
      const float b1 = __shfl_xor_sync(kAll, a1, o), b2 = __shfl_xor_sync(kAll, a2, o);
      a2 = fmaxf(fminf(a1, b1), fmaxf(a2, b2));
      a1 = fmaxf(a1, b1);
    }
    const float g = a2 > -INFINITY ? a1 + a2 : a1;
    if (a.topk_group < a.n_group) {
      // the best groups leave one by one; equal ones leave together and are too many then
      const uint32_t gkey = group < a.n_group ? key_of(g) : 0;
      uint32_t mine = gkey, last = 0;
#pragma unroll 4
      for (int s = 0; s < a.topk_group; ++s) {
        last = __reduce_max_sync(kAll, mine);
        if (mine == last) mine = 0;
      }
      bool in = mine != gkey;
      const float gi = value_of(last), go = value_of(__reduce_max_sync(kAll, mine));
      // Too near to tell apart in fp32, by any group's error? (No group left: go is a NaN.) What a sum
      // is off by goes with the magnitudes of its two choices, which may cancel in it.
      const float mag = fabsf(a1) + (a2 > -INFINITY ? fabsf(a2) : 0.f);
      if (__any_sync(kAll, g > -INFINITY && gi - go <= 2.f * tol * (1.f + mag)) ||
          __popc(__ballot_sync(kAll, in)) != a.topk_group << a.lpg_log2) {
        const float from = second - tol * (1.f + fabsf(second));
        uint32_t two = 0;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
          two |= j < n && !(c[j] < from) ? 1u << j : 0u;
          row_l[warp][lane * NPL + j] = l[j];
        }
        in = group_rank_exact<T>(a, row, top, e0, n, group, two, &row_l[warp][lane * NPL]) <
             a.topk_group;
      }
      if (!in) {
        best = second = -INFINITY;
#pragma unroll
        for (int j = 0; j < NPL; ++j) c[j] = -INFINITY;
      }
    }
  } else {
    best = c[0];
#pragma unroll
    for (int j = 1; j < NPL; ++j) best = fmaxf(best, c[j]);
  }
  // k-th largest of the lanes' largest (GROUPED: two largest, as few lanes are left) choices.
  // Equal ones leave together: the bound only gets lower.
  uint32_t mine = key_of(best), bound = 0;
  uint32_t then = GROUPED ? key_of(second) : 0;
#pragma unroll 4
  for (int s = 0; s < a.topk; ++s) {
    bound = __reduce_max_sync(kAll, mine);
    if (mine == bound) {
      mine = then;
      if (GROUPED) then = 0;
    }
  }
  const float kth = value_of(bound);
  const bool few = !(bound > key_of(-INFINITY));  // fewer than k finite ones among them
  const float limit = kth - tol * (1.f + fabsf(kth));
  uint32_t left = 0;  // this lane's candidates
#pragma unroll
  for (int j = 0; j < NPL; ++j) left |= c[j] >= limit ? 1u << j : 0u;
  if (left) {
    float* pc = &row_c[warp][lane * NPL];
    float* pl = &row_l[warp][lane * NPL];
    if (NPL % 4 == 0) {
#pragma unroll
      for (int j = 0; j + 3 < NPL; j += 4) {
        *reinterpret_cast<float4*>(pc + j) = make_float4(c[j], c[j + 1], c[j + 2], c[j + 3]);
        *reinterpret_cast<float4*>(pl + j) = make_float4(l[j], l[j + 1], l[j + 2], l[j + 3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NPL; ++j) {
        pc[j] = c[j];
        pl[j] = l[j];
      }
    }
  }
  int count = 0;
  for (unsigned m = __ballot_sync(kAll, left != 0); m; m = __ballot_sync(kAll, left != 0)) {
    // the lanes of m put down one candidate each
    if (left) {
      const int slot = count + __popc(m & ((1u << lane) - 1));
      if (slot < 32) place[warp][slot] = lane * NPL + __ffs(left) - 1;
      left &= left - 1;
    }
    count += __popc(m);
  }
  __syncwarp();
  // (fewer than k: the bound is infinity, by a bias, and its limit a NaN)
  if (few || count > 32 || count < a.topk) {
    route_row_exact<T>(a, t, lane);
    return;
  }
  // a candidate for each lane of a run of W lanes, the other runs scan their share for it
  const int W = count <= 8 ? 8 : count <= 16 ? 16 : 32;
  const int ci = lane & (W - 1);
  float choice = -INFINITY, logit = 0.f;
  int id = 0x7fffffff;
  if (ci < count) {
    const int at = place[warp][ci];
    choice = row_c[warp][at];
    logit = row_l[warp][at];
    const int from = at / NPL;
    id = (GROUPED ? (from >> a.lpg_log2) * a.gsz + (from & (a.lpg - 1)) * NPL : from * NPL) + at % NPL;
  }
  const unsigned long long key = (unsigned long long)key_of(choice) << 32 | (uint32_t)~id;
  cand[warp][lane] = lane < count ? key : 0;  // the same trips for all lanes: zeros outrank nobody
  __syncwarp();
  int rank = 0;
  const unsigned long long* other = &cand[warp][lane / W];
#pragma unroll 4
  for (int q = 0; q < count; q += 32 / W) rank += other[q] > key;
  for (int o = W; o < 32; o <<= 1) rank += __shfl_xor_sync(kAll, rank, o);
  if (!plain) {
    // neighbours in the order, the first one out among them, too near to tell apart?
    if (lane < count) sorted[warp][rank] = choice;
    if (lane == 0) sorted[warp][count] = -INFINITY;
    __syncwarp();
    const bool near = lane < count && rank < a.topk &&
                      choice - sorted[warp][rank + 1] <= tol * (1.f + fabsf(choice));
    if (__any_sync(kAll, near)) rank = rank_exact<T>(a, row, top, e0, n, logit, id, count, lane);
  }
  const bool chosen = lane < count && rank < a.topk;
  float w = chosen ? score(logit) : 0.f;
  if (a.renorm) w = __fdividef(w, fmaxf(warp_sum(w), 1e-20f));
  if (chosen) {
    a.topw[t * a.topk + rank] = w * a.scale;
    a.topi[t * a.topk + rank] = id;
  }
}

template <typename T, int NPL>
void launch_npl(const RouteArgs& a, cudaStream_t st) {
  const int grid = (a.T + kWarps - 1) / kWarps;
  auto fn = a.softmax ? (a.n_group > 1 ? route_topk_kernel<T, NPL, true, true>
                                       : route_topk_kernel<T, NPL, true, false>)
                      : (a.n_group > 1 ? route_topk_kernel<T, NPL, false, true>
                                       : route_topk_kernel<T, NPL, false, false>);
  fn<<<grid, kWarps * 32, 0, st>>>(a);
}

template <typename T>
int launch_route(const RouteArgs& a, cudaStream_t st) {
  switch (a.npl) {
    case 1: launch_npl<T, 1>(a, st); break;
    case 2: launch_npl<T, 2>(a, st); break;
    case 4: launch_npl<T, 4>(a, st); break;
    case 8: launch_npl<T, 8>(a, st); break;
    case 16: launch_npl<T, 16>(a, st); break;
    default: launch_npl<T, 32>(a, st); break;
  }
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
  if (T < 0 || T > kMaxRows || E < 1 || topk < 1 || topk > 32 || topk > E)
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
  a.lpg_log2 = 5;
  while (a.lpg * n_group > 32) {
    a.lpg >>= 1;
    --a.lpg_log2;
  }
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
