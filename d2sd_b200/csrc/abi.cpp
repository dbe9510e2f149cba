// ABI-level helpers: version, thread-local last error, device SM count, calls with
// packed arguments.
#include <cuda_runtime.h>
#include <string.h>

#include <mutex>
#include <string>
#include <type_traits>
#include <utility>

#include "../../include/d2sd.h"

namespace d2sd {

namespace {
thread_local std::string g_last_error;
}

void set_last_error(const std::string& msg) { g_last_error = msg; }

int current_sm_count() {
  static int cache[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (cache[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
      n = 148;
    cache[dev] = n;
  }
  return cache[dev];
}

namespace {
// An argument out of its word: pointers and integers as an int64, a float as a double.
template <typename A>
A unpack(const int64_t& word) {
  if constexpr (std::is_pointer<A>::value) {
    return reinterpret_cast<A>(static_cast<intptr_t>(word));
  } else if constexpr (std::is_floating_point<A>::value) {
    double d;
    memcpy(&d, &word, sizeof(d));
    return static_cast<A>(d);
  } else {
    return static_cast<A>(word);
  }
}
template <typename... A, size_t... I>
int call(int (*fn)(A...), const int64_t* words, std::index_sequence<I...>) {
  return fn(unpack<A>(words[I])...);
}
template <typename... A>
int call(int (*fn)(A...), const int64_t* words, int32_t num_words) {
  if (num_words != static_cast<int32_t>(sizeof...(A))) {
    set_last_error("d2sd_call: wrong number of arguments");
    return D2SD_ERR_INVALID_ARGUMENT;
  }
  return call(fn, words, std::index_sequence_for<A...>());
}
}  // namespace

}  // namespace d2sd

extern "C" int d2sd_call(int32_t entry, const void* words, int32_t num_words) {
  using namespace d2sd;
  const int64_t* w = static_cast<const int64_t*>(words);
  switch (w ? entry : -1) {
    case D2SD_CALL_APPEND_KV: return call(&d2sd_append_kv, w, num_words);
    case D2SD_CALL_READ_KV: return call(&d2sd_read_kv, w, num_words);
    case D2SD_CALL_PAGED_ATTENTION: return call(&d2sd_paged_attention, w, num_words);
  }
  set_last_error("d2sd_call: unknown entry");
  return D2SD_ERR_INVALID_ARGUMENT;
}

extern "C" int d2sd_version(void) { return 100; }

extern "C" const char* d2sd_last_error(void) { return d2sd::g_last_error.c_str(); }
