// Packed forms of entry points that are called at a few tokens, where the host's conversion of one
// argument after another is a good part of a call (ctypes: 0.1 us each, 1.8 to 2.1 us for 16 to 21
// of them; 0.5 us packed). The words are the arguments of the entry of the same name, in order.
#include <string.h>

#include <tuple>
#include <type_traits>
#include <utility>

#include "fusion_b200.h"
#include "host_util.h"

namespace fus {
namespace {

struct Words {
  const unsigned char* p;
  int bad = -1;  // the first argument that does not fit its type

  template <typename A>
  A take(int i) {
    static_assert(sizeof(A) <= 8, "one word for an argument");
    if constexpr (std::is_same_v<A, float>) {
      double d;
      memcpy(&d, p + 8 * i, 8);
      return (float)d;
    } else if constexpr (std::is_same_v<A, int>) {
      long v;
      memcpy(&v, p + 8 * i, 8);
      if (v != (long)(int)v && bad < 0) bad = i;
      return (int)v;
    } else {
      A v;
      memcpy(&v, p + 8 * i, 8);
      return v;
    }
  }
};

template <typename... A, size_t... I>
int call_packed(const char* name, int (*fn)(A...), const void* words, std::index_sequence<I...>) {
  if (!words) return set_error(FUS_E_INVALID, "%s: null words", name);
  Words w{reinterpret_cast<const unsigned char*>(words)};
  std::tuple<A...> args{w.take<A>((int)I)...};
  if (w.bad >= 0) return set_error(FUS_E_INVALID, "%s: argument %d out of range", name, w.bad);
  return fn(std::get<I>(args)...);
}

template <typename... A>
int call_packed(const char* name, int (*fn)(A...), const void* words) {
  return call_packed(name, fn, words, std::index_sequence_for<A...>{});
}

}  // namespace
}  // namespace fus

extern "C" int fus_norm_gate_residual_packed(const void* words) {
  return fus::call_packed("norm_gate_residual", fus_norm_gate_residual, words);
}
extern "C" int fus_route_topk_packed(const void* words) {
  return fus::call_packed("route_topk", fus_route_topk, words);
}
extern "C" int fus_fp4_quantize_packed(const void* words) {
  return fus::call_packed("fp4_quantize", fus_fp4_quantize, words);
}
extern "C" int fus_fp4_dequantize_packed(const void* words) {
  return fus::call_packed("fp4_dequantize", fus_fp4_dequantize, words);
}
extern "C" int fus_fp4_expert_gemm_packed(const void* words) {
  return fus::call_packed("fp4_expert_gemm", fus_fp4_expert_gemm, words);
}
