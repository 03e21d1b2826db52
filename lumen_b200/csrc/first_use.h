// Set-up that a process does once per device and key.
#pragma once
#include <mutex>
#include <set>
#include <utility>

namespace lb {

class FirstUse {
    std::mutex mutex_;
    std::set<std::pair<int, const void*>> done_;

public:
    // Runs `setup` unless it has been run for this device and key. Calls that come meanwhile wait for it, so that all of them find it done when this
    // returns; one that throws leaves it to the next.
    template <class F>
    void run(int device, const void* key, F setup) {
        std::lock_guard<std::mutex> lock(mutex_);
        if (done_.count({device, key})) return;
        setup();
        done_.insert({device, key});
    }
};

}  // namespace lb
