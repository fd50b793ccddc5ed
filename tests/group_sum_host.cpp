// csrc/group_sum.hpp on the CPU: a thread a lane, barriers for the wave and the workgroup, and one wave that is late:
// after each workgroup barrier it goes on only when all others stand at the next one or have ended, so that whatever
// they write too early is there when it reads.  The values are small whole numbers, whose sums are exact; prints the
// number of wrong sums.
#include <array>
#include <atomic>
#include <barrier>
#include <chrono>
#include <cstdio>
#include <memory>
#include <thread>
#include <vector>

#define __device__
#define __forceinline__ inline

namespace emulated {
struct Index {
    int x;
};
thread_local Index thread;
int slow_wave = 0;

struct Wave {
    std::barrier<> meet{64};
    std::array<float, 64> at{};
};
std::vector<std::unique_ptr<Wave>> waves;
std::unique_ptr<std::barrier<>> group;
std::atomic<int> arrived{0};  // at workgroup barriers, or ended (once for each of kMany barriers), the lanes of the others
thread_local int passed = 0;
constexpr int kMany = 1 << 16;

// f(the 64 lanes' values, this lane)
template <class F>
float exchange(float v, F&& f) {
    Wave& w = *waves[thread.x / 64];
    const int lane = thread.x % 64;
    w.at[lane] = v;
    w.meet.arrive_and_wait();
    const float got = f(w.at, lane);
    w.meet.arrive_and_wait();
    return got;
}
}  // namespace emulated

#define threadIdx emulated::thread

inline float __shfl_xor(float v, int by) {
    return emulated::exchange(v, [&](const auto& at, int lane) { return at[lane ^ by]; });
}
inline void __syncthreads() {
    const bool late = emulated::thread.x / 64 == emulated::slow_wave;
    if (!late) ++emulated::arrived;
    emulated::group->arrive_and_wait();
    ++emulated::passed;
    const int others = 64 * (static_cast<int>(emulated::waves.size()) - 1);
    while (late && emulated::arrived < others * (emulated::passed + 1))
        std::this_thread::sleep_for(std::chrono::microseconds(200));
}

namespace smx {
inline float row_total(float v) {
    return emulated::exchange(v, [](const auto& at, int lane) {
        float s = 0.0f;
        for (int i = 0; i < 16; ++i) s += at[lane / 16 * 16 + i];
        return s;
    });
}
}  // namespace smx

#include "group_sum.hpp"

namespace {

using namespace smx::node;

constexpr int kRows = 6;

int value(int row, int k, int lane) { return (row * 131 + k * 17 + lane * (lane + row) * (k + 1)) % 61; }

float total(int row, int k, int lanes) {
    int s = 0;
    for (int i = 0; i < lanes; ++i) s += value(row, k, i);
    return static_cast<float>(s);
}

template <int G, int K, class S>
int one_sum(int row, int first, S&& sum) {
    float v[K];
    for (int k = 0; k < K; ++k) v[k] = static_cast<float>(value(row, first + k, threadIdx.x));
    sum(v);
    int wrong = 0;
    for (int k = 0; k < K; ++k) wrong += v[k] != total(row, first + k, G);
    return wrong;
}

// The wrong sums of all lanes, with each wave in turn the late one.
template <int G, class F>
int wrong_sums(F&& rows) {
    int wrong = 0;
    emulated::waves.clear();
    for (int w = 0; w < G / 64; ++w) emulated::waves.push_back(std::make_unique<emulated::Wave>());
    for (emulated::slow_wave = 0; emulated::slow_wave < G / 64; ++emulated::slow_wave) {
        emulated::group = std::make_unique<std::barrier<>>(G);
        emulated::arrived = 0;
        std::vector<int> of(G);
        std::vector<std::thread> lanes;
        for (int t = 0; t < G; ++t)
            lanes.emplace_back([&, t] {
                threadIdx.x = t;
                of[t] = rows();
                if (t / 64 != emulated::slow_wave) emulated::arrived += emulated::kMany;
            });
        for (auto& t : lanes) t.join();
        for (int n : of) wrong += n;
    }
    return wrong;
}

template <int G>
int check() {
    typename GradientSums<G>::Room room{};
    typename GroupSum<G, 1>::Room other{};
    // a gradient's rows: both rounds, then the second alone (no d)
    int wrong = wrong_sums<G>([&] {
        GradientSums<G> sums{room};
        int n = 0;
        for (int r = 0; r < kRows; ++r) {
            n += one_sum<G, 1>(r, 0, [&](float(&v)[1]) { sums.sum(v); });
            n += one_sum<G, 5>(r, 1, [&](float(&v)[5]) { sums.sum(v); });
        }
        return n;
    });
    wrong += wrong_sums<G>([&] {
        GradientSums<G> sums{room};
        int n = 0;
        for (int r = 0; r < kRows; ++r) n += one_sum<G, 5>(r, 1, [&](float(&v)[5]) { sums.sum(v); });
        return n;
    });
    // a forward call's rows: the same sum twice
    wrong += wrong_sums<G>([&] {
        int turn = 0, n = 0;
        for (int r = 0; r < 2 * kRows; ++r) n += one_sum<G, 1>(r, 0, [&](float(&v)[1]) { GroupSum<G, 1>::sum(v, other, turn); });
        return n;
    });
    std::printf("%d lanes: %d wrong\n", G, wrong);
    return wrong;
}

}  // namespace

int main() { return check<128>() + check<256>() ? 1 : 0; }
