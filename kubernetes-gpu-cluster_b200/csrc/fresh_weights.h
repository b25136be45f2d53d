// On which streams weights have been written that no later launch has waited for in full.  Products read weights before they wait for the kernel before them
// (programmatic dependent launch); what the writer left is certain to be seen only behind an ordinary launch, so the first product on the writer's stream is one,
// whichever thread makes it and whatever else was launched in between, there or elsewhere.
#pragma once
#include <stdint.h>

#include <atomic>
#include <mutex>
#include <thread>
#include <vector>

namespace kge {
class FreshWeights {
 public:
  // `stream`: a cudaStream_t.  0 and 1 are the legacy stream; 2 is the calling thread's own, a stream of its own in each.
  void written(const void* stream) {
    const Key k = key(stream);
    std::lock_guard<std::mutex> lock(m_);
    for (const Key& o : streams_)
      if (o == k) return;
    try {
      streams_.push_back(k);
    } catch (...) {                              // (callers are C: without room for it, every stream's products are ordinary from now on)
      all_ = true;
    }
    some_.store(true, std::memory_order_release);
  }
  // Whether a product on `stream` has to be an ordinary launch; asked once for a launch that then is.  capturing(): whether the stream records a graph, whose
  // launches order nothing for what is launched after the recording; asked only where it matters.
  template <typename F>
  bool take(const void* stream, F capturing) {
    if (!some_.load(std::memory_order_acquire)) return false;
    const Key k = key(stream);
    std::lock_guard<std::mutex> lock(m_);
    for (size_t i = 0; i < streams_.size(); ++i)
      if (streams_[i] == k) {
        if (!capturing()) {
          streams_[i] = streams_.back();
          streams_.pop_back();
          some_.store(all_ || !streams_.empty(), std::memory_order_release);
        }
        return true;
      }
    return all_;
  }

 private:
  struct Key {
    uintptr_t stream;
    std::thread::id thread;
    bool operator==(const Key& o) const { return stream == o.stream && thread == o.thread; }
  };
  static Key key(const void* stream) {
    const uintptr_t s = (uintptr_t)stream;
    return Key{s == 1 ? 0 : s, s == 2 ? std::this_thread::get_id() : std::thread::id()};
  }
  std::mutex m_;
  std::vector<Key> streams_;                     // few: an entry stays until its stream's next product, once for a stream
  bool all_ = false;
  std::atomic<bool> some_{false};
};
}  // namespace kge
