// Set-up that is needed once on every device, such as a kernel's shared-memory limit (an attribute of the function on the
// device that is current). A failure is not remembered: the next call tries again.
#pragma once
#include <mutex>
#include <set>

namespace gpt {

class DeviceOnce {
    std::mutex mu_;
    std::set<int> done_;

public:
    template <class F>
    void run(int device, F&& set_up) {
        std::lock_guard<std::mutex> lock(mu_);
        if (done_.count(device)) return;
        set_up();
        done_.insert(device);
    }
};

}  // namespace gpt
