// A positive number that each device has one of, asked for until it is known: an answer of 0 or less (the question failed) is not kept, and one device's says nothing of another's.
#pragma once
#include <atomic>

class LcuPerDevice {
    static constexpr int MOST = 64;
    std::atomic<long long> known[MOST] = {};

public:
    // ask(device): the number; unknown: what is given for a device whose number is not to be had.
    template <class Ask>
    long long get(int device, Ask ask, long long unknown) {
        if (device < 0 || device >= MOST) return unknown;
        long long n = known[device].load(std::memory_order_relaxed);
        if (n == 0) {
            n = ask(device);
            if (n <= 0) return unknown;
            known[device].store(n, std::memory_order_relaxed);
        }
        return n;
    }
};
