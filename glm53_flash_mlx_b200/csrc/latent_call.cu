// glm53_latent_call: the latent-attention entry points from one array of words.
#include <cstring>
#include <tuple>
#include <type_traits>

#include "common.cuh"

namespace {

struct Words {
  const uint64_t* at;
  template <typename T>
  T next() {
    const uint64_t w = *at++;
    if constexpr (std::is_pointer<T>::value) {
      return reinterpret_cast<T>(static_cast<uintptr_t>(w));
    } else if constexpr (std::is_floating_point<T>::value) {
      double d;
      std::memcpy(&d, &w, sizeof(d));
      return static_cast<T>(d);
    } else {
      return static_cast<T>(static_cast<int64_t>(w));
    }
  }
};

// Braced initialisers evaluate in order, which function arguments need not.
template <typename... A>
struct Call {
  std::tuple<A...> args;
  explicit Call(Words w) : args{w.next<A>()...} {}
};
template <typename... A>
int call(int (*fn)(A...), const void* words) {
  Call<A...> c(Words{static_cast<const uint64_t*>(words)});
  return std::apply(fn, c.args);
}

}  // namespace

extern "C" int glm53_latent_call(int entry, const void* words) {
  if (!words || ((uintptr_t)words & 7)) {
    glm53::set_last_error("glm53_latent_call: the words must be non-NULL and 8-byte aligned");
    return GLM53_ERR_INVALID;
  }
  switch (entry) {
    case GLM53_LATENT_PLAN_PAGES: return call(glm53_plan_pages, words);
    case GLM53_LATENT_CACHE_WRITE: return call(glm53_latent_cache_write, words);
    case GLM53_LATENT_ABSORBED: return call(glm53_latent_absorbed, words);
    case GLM53_LATENT_EXPANDED: return call(glm53_latent_expanded, words);
  }
  glm53::set_last_error("glm53_latent_call: no entry point %d", entry);
  return GLM53_ERR_INVALID;
}
