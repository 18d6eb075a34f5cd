/* Two host threads that first ask for different sizes of shared memory at the
 * same time, the larger one delayed between setting the attribute and noting
 * it: what is noted must not be above what is set.  Exit status 0 if so. */
#include "tb_shared_limit.h"

#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <thread>

int main() {
    tb_learn::SharedLimit limit;
    std::mutex m;
    std::condition_variable changed;
    size_t attribute = 0; /* as the CUDA driver would hold it */
    bool large_set = false, small_done = false;
    const auto set = [&](size_t bytes) {
        std::unique_lock<std::mutex> hold(m);
        attribute = bytes;
        if (bytes == 100) {
            large_set = true;
            changed.notify_all(); /* let the other in, if it can come in */
            changed.wait_for(hold, std::chrono::milliseconds(300), [&] { return small_done; });
        }
        return true;
    };
    std::thread large([&] { limit.raise(100, set); });
    {
        std::unique_lock<std::mutex> hold(m);
        changed.wait(hold, [&] { return large_set; });
    }
    std::thread small([&] {
        limit.raise(60, set);
        std::lock_guard<std::mutex> hold(m);
        small_done = true;
        changed.notify_all();
    });
    large.join();
    small.join();
    limit.raise(90, set); /* allowed already, or set now */
    std::printf("attribute %zu\n", attribute);
    if (attribute < 90) return 1;
    tb_learn::SharedLimit refused;
    if (refused.raise(10, [](size_t) { return false; })) return 2; /* not noted where it was refused */
    return refused.raise(10, [](size_t) { return true; }) ? 0 : 3;
}
