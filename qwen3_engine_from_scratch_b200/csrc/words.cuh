// Arguments of a C entry as an array of 64-bit words.
#pragma once

#include <cstdint>
#include <cstring>

namespace b200host {

struct Words {
  const int64_t* word;
  bool fit = true;  // every integer() so far was one

  template <typename T = void>
  T* pointer(int i) const {
    return reinterpret_cast<T*>(static_cast<uintptr_t>(word[i]));
  }
  int64_t wide(int i) const { return word[i]; }
  int integer(int i) {
    const int v = static_cast<int>(word[i]);
    fit = fit && v == word[i];
    return v;
  }
  float real(int i) const {
    double v;
    std::memcpy(&v, word + i, sizeof v);
    return static_cast<float>(v);
  }
};

}  // namespace b200host
