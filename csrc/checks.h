// Argument checks whose messages carry names and numbers. The text is put together with
// std::string alone: TORCH_CHECK formats several arguments through a std::ostringstream, which in an
// extension that runs beside another libstdc++ than the one it was compiled with ends the process
// instead of raising (seen with the pip builds of torch).
#pragma once
#include <string>
#include <torch/extension.h>

namespace appcorr {
inline std::string check_text(const char* s) { return s; }
inline std::string check_text(int64_t v) { return std::to_string(v); }
template <typename... A>
std::string check_message(const A&... parts) {
  std::string s;
  ((s += check_text(parts)), ...);
  return s;
}
}  // namespace appcorr

#define APPCORR_CHECK(cond, ...) TORCH_CHECK(cond, ::appcorr::check_message(__VA_ARGS__))
