// PerDeviceOnce without a device: what a failure leaves, and two threads on their first call.
#include <chrono>
#include <cstdio>
#include <future>

#include "../../tensorlib_b200/csrc/common.cuh"

#define EXPECT(cond)                                          \
    do {                                                      \
        if (!(cond)) {                                        \
            std::printf("FAIL line %d: %s\n", __LINE__, #cond); \
            return 1;                                         \
        }                                                     \
    } while (0)

int main() {
    {
        tlb::PerDeviceOnce once;
        int calls = 0;
        auto fails = [&] { calls++; return cudaErrorInvalidValue; };
        auto works = [&] { calls++; return cudaSuccess; };
        EXPECT(once.run_on(3, fails) == cudaErrorInvalidValue && calls == 1);
        EXPECT(once.run_on(3, fails) == cudaErrorInvalidValue && calls == 2);      // tried again
        EXPECT(once.run_on(3, works) == cudaSuccess && calls == 3);
        EXPECT(once.run_on(3, fails) == cudaSuccess && calls == 3);                // done
        EXPECT(once.run_on(4, works) == cudaSuccess && calls == 4);                // another device
        for (int i = 0; i < 2; i++) EXPECT(once.run_on(64, works) == cudaSuccess && calls == 5 + i);   // beyond the mask: every time
    }
    {
        // The first thread is held inside its setting until the second's call has returned: that one must have set the attributes
        // itself. The wait has an end, so that a second thread that waits for the first shows as a failure.
        tlb::PerDeviceOnce once;
        std::promise<void> inside, returned;
        std::shared_future<void> second = returned.get_future().share();
        bool in_time = false, by_second = false;
        auto first = std::async(std::launch::async, [&] {
            return once.run_on(0, [&] {
                inside.set_value();
                in_time = second.wait_for(std::chrono::seconds(10)) == std::future_status::ready;
                return cudaSuccess;
            });
        });
        inside.get_future().wait();
        EXPECT(once.run_on(0, [&] { by_second = true; return cudaSuccess; }) == cudaSuccess);
        returned.set_value();
        EXPECT(first.get() == cudaSuccess && in_time && by_second);
    }
    std::printf("OK attributes\n");
    return 0;
}
