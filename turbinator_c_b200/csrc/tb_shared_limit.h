/*
 * What a kernel has been allowed of dynamic shared memory on a device.  Host
 * threads that first ask for different sizes at the same time must not leave
 * the lower one set and the higher one noted, so sizes are set one after the
 * other and only ever grow; what is allowed already takes no lock.
 */
#ifndef TB_SHARED_LIMIT_H
#define TB_SHARED_LIMIT_H

#include <stddef.h>

#include <atomic>
#include <mutex>

namespace tb_learn {

inline std::mutex shared_limit_lock;

class SharedLimit {
    std::atomic<size_t> allowed_{0};

  public:
    /* Whether `bytes` are allowed, by set(bytes) where they were not yet. */
    template <class Set> bool raise(size_t bytes, Set &&set) {
        if (bytes <= allowed_.load(std::memory_order_acquire)) return true;
        std::lock_guard<std::mutex> hold(shared_limit_lock);
        if (bytes <= allowed_.load(std::memory_order_relaxed)) return true;
        if (!set(bytes)) return false;
        allowed_.store(bytes, std::memory_order_release);
        return true;
    }
};

} /* namespace tb_learn */

#endif
