// A handle's workspaces: device memory that its launches use between their kernels, one for each stream.
#ifndef TETRIS_CSRC_WORKSPACE_H_
#define TETRIS_CSRC_WORKSPACE_H_

#include <algorithm>
#include <exception>

#include "common.h"

namespace tetris {

// A number of the calling thread, never given to another one.
inline uint64_t thread_number() {
  static std::atomic<uint64_t> threads{0};
  static thread_local const uint64_t mine = ++threads;
  return mine;
}

class Workspaces {
 public:
  // That of the stream, at least `need` bytes.  A buffer that has to grow is replaced and kept until the handle goes: a
  // captured graph may hold its address.  It at least doubles, so that those kept are together no larger than the last one.
  int get(hipStream_t stream, size_t need, uint8_t** out) {
    *out = nullptr;
    if (!need) return TETRIS_OK;
    try {
      std::lock_guard<std::mutex> lock(mu_);
      Space& s = space_[{stream, stream == hipStreamPerThread ? thread_number() : 0}];
      if (s.bytes < need) {
        hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing(stream, &cap) == hipSuccess && cap != hipStreamCaptureStatusNone)
          return fail(TETRIS_EINVAL, "this launch would allocate its workspace: prepare it before capturing");
        retired_.reserve(retired_.size() + 1);
        void* d = nullptr;
        size_t bytes = std::max(need, 2 * s.bytes);
        if (bytes > need && hipMalloc(&d, bytes) != hipSuccess) {
          (void)hipGetLastError();  // no room for twice as much
          d = nullptr;
        }
        if (!d) TETRIS_HIP(hipMalloc(&d, bytes = need));
        if (s.ptr) retired_.push_back(s.ptr);
        s.ptr = d;
        s.bytes = bytes;
      }
      *out = static_cast<uint8_t*>(s.ptr);
      return TETRIS_OK;
    } catch (const std::exception& e) {
      return fail(TETRIS_EINVAL, "%s", e.what());
    }
  }
  void release() {
    for (auto& s : space_)
      if (s.second.ptr) (void)hipFree(s.second.ptr);
    for (void* p : retired_) (void)hipFree(p);
    space_.clear();
    retired_.clear();
  }

 private:
  struct Space { void* ptr = nullptr; size_t bytes = 0; };
  std::mutex mu_;
  std::map<std::pair<hipStream_t, uint64_t>, Space> space_;  // the number: of the thread, for hipStreamPerThread, which is one value for many streams
  std::vector<void*> retired_;  // replaced by larger ones; a captured graph may hold their addresses
};

}  // namespace tetris

#endif  // TETRIS_CSRC_WORKSPACE_H_
