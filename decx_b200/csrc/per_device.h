// A number that is asked for once per device and kept.  A query that fails (0 or less) is not kept: the next call asks again.
// Plain C++, so that it can be checked without a GPU.
#pragma once
#include <atomic>

namespace dxb_host {

class PerDevice {
  public:
    template <typename Ask>
    int get(int device, Ask&& ask) {
        if (device < 0 || device >= DEVICES) return ask();
        int n = known_[device].load(std::memory_order_relaxed);
        if (n == 0) {
            n = ask();
            if (n > 0) known_[device].store(n, std::memory_order_relaxed);
        }
        return n;
    }

  private:
    static constexpr int DEVICES = 64;
    std::atomic<int> known_[DEVICES] = {};
};

}  // namespace dxb_host
