// pkv_call: an entry point with its arguments packed into 8-byte words (host code only).
#include <cstring>
#include <type_traits>
#include <utility>
#include "common.h"
#include "../../include/pagedkv.h"

namespace {

template <typename A>
A word(const char* p) {
  if constexpr (std::is_floating_point<A>::value) {
    double x;
    std::memcpy(&x, p, 8);
    return (A)x;
  } else {
    int64_t x;
    std::memcpy(&x, p, 8);
    return (A)x;  // (pointers: as wide)
  }
}
template <typename... A, size_t... I>
int unpack(int (*f)(A...), const char* p, std::index_sequence<I...>) {
  return f(word<A>(p + 8 * I)...);
}
template <typename... A>
int call(int (*f)(A...), const void* words, int32_t count) {
  return count == (int32_t)sizeof...(A) ? unpack(f, (const char*)words, std::index_sequence_for<A...>{}) : (int)pkv::kBadArg;
}

}  // namespace

extern "C" int pkv_call(int32_t entry, const void* words, int32_t count) {
  if (!words) return pkv::kBadArg;
  switch (entry) {
    case PKV_CALL_APPEND_FP8: return call(pkv_append_paged_kv_cache_fp8, words, count);
    case PKV_CALL_NORM_ROPE: return call(pkv_append_paged_kv_cache_norm_rope, words, count);
    case PKV_CALL_READ_FP8: return call(pkv_read_paged_kv_cache_fp8, words, count);
    case PKV_CALL_DECODE_FP8: return call(pkv_batch_decode_fp8, words, count);
  }
  return pkv::kBadArg;
}
