"""The search in a row's histogram of logits (csrc/sample_search.h), run on the host with a thread for every one of a workgroup's."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

HOST = '''
#include <pthread.h>
#include <unistd.h>
#include <atomic>
#include <cstdio>
#include <thread>
#include <vector>
#define __device__
#define __forceinline__ inline
struct Index { unsigned x; };
static thread_local Index threadIdx;
static pthread_barrier_t barrier;
static void __syncthreads() { pthread_barrier_wait(&barrier); }
#include "sample_search.h"
using namespace afhip;
'''


def run(tmp_path, body):
    source, binary = tmp_path / "search.cpp", tmp_path / "search"
    source.write_text(HOST + body)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-Wall", "-Werror", "-I", os.path.join(ROOT, "antfly_amd", "csrc"), str(source), "-o", str(binary)],
                   check=True)
    done = subprocess.run([str(binary)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout


def test_one_search_after_the_other(tmp_path):
    """Every thread gets every search's bin, however late it comes to read it: searches may follow one another at once."""
    run(tmp_path, '''
// A number in LDS that all wavefronts but the first read late.
struct Late {
    std::atomic<uint32_t> held{0};
    void operator=(uint32_t v) { held = v; }
    operator uint32_t() {
        if (threadIdx.x >= 64) usleep(20000);
        return held;
    }
};
struct Shared {
    uint32_t counts[kSampleBins];
    unsigned long long sums[kSampleBins];
    Late found_bin;
} s;
int main() {
    for (uint32_t b = 0; b < kSampleBins; ++b) {  // three tokens of weight 5 a bin
        s.counts[b] = 3 * b;
        s.sums[b] = 15 * b;
    }
    pthread_barrier_init(&barrier, nullptr, kSampleThreads);
    const Target targets[] = {{3 * 700 + 1, 0}, {0, 15 * 40 + 1}, {0, 15 * 40}, {0, 15 * 1023 + 1}, {0, 1000000000}, {1, 0}};
    const uint32_t bins[] = {700, 40, 39, 1023, kSampleBins, 0};
    std::atomic<int> wrong{0};
    std::vector<std::thread> threads;
    for (int t = 0; t < kSampleThreads; ++t) {
        threads.emplace_back([&, t] {
            threadIdx.x = t;
            for (int i = 0; i < 6; ++i) wrong += find_bin(targets[i], 0, 0, 3 * kSampleBins, 15 * kSampleBins, s) != bins[i];
        });
    }
    for (auto& t : threads) t.join();
    if (wrong != 0) std::printf("%d of the threads' bins are wrong\\n", wrong.load());
    return wrong != 0;
}
''')
