// What a launcher sets up once on each device (host side).  Launchers are called from several threads at a time: their first calls wait for the one
// that sets up, nobody launches before it is done, and a set-up that failed is tried again by the next call.
#pragma once
#include <atomic>
#include <mutex>

struct FgPerDevice {
    std::atomic<bool> done[64];
    std::mutex busy;
};
// 0, or the code that `set_up` returned
template <typename F>
static inline int fg_set_up_on(FgPerDevice &s, int device, F set_up) {
    const bool kept = device >= 0 && device < 64;
    if (kept && s.done[device].load(std::memory_order_acquire)) return 0;
    std::lock_guard<std::mutex> alone(s.busy);
    if (kept && s.done[device].load(std::memory_order_relaxed)) return 0;
    const int code = (int)set_up();
    if (kept && code == 0) s.done[device].store(true, std::memory_order_release);
    return code;
}
