// Refusals of an entry point's arguments: a Python ValueError, or a RuntimeError where the older entry points raise one.
// The text is put together without streams: those of an extension that links its own libstdc++ statically crash on numbers.
#pragma once

#include <pybind11/pybind11.h>

#include <string>
#include <type_traits>

namespace rad {

inline std::string text_of(const char* s) { return s; }
template <typename N, typename = std::enable_if_t<std::is_integral<N>::value>>
std::string text_of(N n) { return std::to_string(n); }

template <typename... A>
std::string text_all(const A&... parts) {
  return (std::string() + ... + text_of(parts));
}

template <typename... A>
[[noreturn]] void refuse_value(const A&... why) {
  throw pybind11::value_error(text_all(why...));
}

}  // namespace rad

#define RAD_CHECK_VALUE(ok, ...) \
  do {                           \
    if (!(ok)) ::rad::refuse_value(__VA_ARGS__); \
  } while (0)
