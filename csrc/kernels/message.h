// Numbers, shapes and devices as text for error messages. They are made without
// C++ streams: where the extension carries a C++ runtime of its own next to
// PyTorch's (a static libstdc++), formatting a number through a stream can crash
// instead of raising.
#pragma once
#include <torch/extension.h>

#include <string>

namespace nk {

inline std::string num(int64_t n) { return std::to_string(n); }

inline std::string dims(const torch::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

inline std::string place(const torch::Tensor& t) { return t.device().str(); }

inline const char* type_name(const torch::Tensor& t) { return c10::toString(t.scalar_type()); }

}  // namespace nk
