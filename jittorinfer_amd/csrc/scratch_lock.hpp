// Locks of scratch areas, one of 256 by an area's address.
#pragma once

#include <stdint.h>

#include <mutex>

namespace mla {

// Areas are allocations of the device's allocator, aligned to 512 bytes and, large ones, to 2 MB: what tells them apart are the address's upper bits, all of
// which a multiplication by 2^64 over the golden ratio carries into its top byte (Fibonacci hashing).
inline unsigned scratch_lock_index(const void * area) { return (unsigned) (((uint64_t) (uintptr_t) area >> 9) * 0x9e3779b97f4a7c15ull >> 56); }

// Held while a launch of several kernels that hand each other scratch is queued; no area, nothing held.
class ScratchLock {
    std::unique_lock<std::mutex> held;

  public:
    explicit ScratchLock(const void * area) {
        static std::mutex locks[256];
        if (area) held = std::unique_lock<std::mutex>(locks[scratch_lock_index(area)]);
    }
};

}  // namespace mla
