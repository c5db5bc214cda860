// What a kernel needs once on each device before its first launch there:
// function attributes, a check of what the compiler made of it.  Host only.
#pragma once

#include <stdint.h>

#include <atomic>

namespace s2 {

// Runs set_up unless it has succeeded for this device before, and returns its
// result (zero: success, of whatever type).  Only a success is remembered, and
// only once it is complete: after a failure the next call tries and fails
// again, and a thread that finds the device set up finds all of it done.  Two
// threads may run set_up at once; it has to bear that, as setting an attribute
// twice does.
template <class F>
auto set_up_once(std::atomic<uint64_t>& done, int device, F set_up) -> decltype(set_up())
{
    const uint64_t bit = device >= 0 && device < 64 ? 1ull << device : 0; // others each time
    if (done.load(std::memory_order_acquire) & bit) return decltype(set_up())(0);
    const auto r = set_up();
    if (r == decltype(set_up())(0)) done.fetch_or(bit, std::memory_order_release);
    return r;
}

} // namespace s2
