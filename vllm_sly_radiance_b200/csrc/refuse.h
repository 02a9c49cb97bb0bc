// Refusals of an entry point's arguments: a Python ValueError.
// The text is put together without streams: those of an extension that links its own libstdc++ statically crash on numbers.
#pragma once

#include <pybind11/pybind11.h>

#include <string>

namespace rad {

inline std::string text_of(const char* s) { return s; }
inline std::string text_of(long long n) { return std::to_string(n); }
inline std::string text_of(int64_t n) { return std::to_string(n); }
inline std::string text_of(int n) { return std::to_string(n); }

template <typename... A>
[[noreturn]] void refuse_value(const A&... why) {
  throw pybind11::value_error((std::string() + ... + text_of(why)));
}

}  // namespace rad

#define RAD_CHECK_VALUE(ok, ...) \
  do {                           \
    if (!(ok)) ::rad::refuse_value(__VA_ARGS__); \
  } while (0)
