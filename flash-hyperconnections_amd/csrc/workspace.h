// Scratch memory of a call, in pieces.
#pragma once

#include <cstdint>

namespace fh {

// Takes pieces of a workspace; without one it only adds up their sizes.
class Workspace {
 public:
  explicit Workspace(void* base) : base_(static_cast<char*>(base)) {}
  template <typename E>
  E* take(int64_t count) {
    const int64_t at = used_;
    used_ += (count * static_cast<int64_t>(sizeof(E)) + 255) / 256 * 256;
    return base_ != nullptr ? reinterpret_cast<E*>(base_ + at) : nullptr;
  }
  bool dry() const { return base_ == nullptr; }
  int64_t used() const { return used_; }

 private:
  char* base_;
  int64_t used_ = 0;
};

}  // namespace fh
