// Calls from several threads on shared streams, with the entry points as they are
// (csrc/q4rdna_layer.cpp, csrc/q4rdna_branch.cpp) and stand-ins for HIP and for the
// kernels' launches, which look at what the launches of a call need of each other:
// the call's scratch, from its first launch to its last, is no other call's.
// Built by the Makefile next to this file with AddressSanitizer and
// UndefinedBehaviorSanitizer, run by tests/test_scratch_threads.py.  No GPU is used.
//
// Device memory is the host's here, and a launch writes its number into the
// scratch that it was given, waits a little, and looks whether it is still there.
#include <atomic>
#include <chrono>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <thread>
#include <vector>

#include "q4rdna_layer_host.h"

namespace {

std::atomic<int> g_failures{0}, g_launches{0}, g_side_by_side{0}, g_inside{0};
std::atomic<uint32_t> g_next{1};

void rest() { std::this_thread::sleep_for(std::chrono::microseconds(200)); }

// A launch that has the scratch at `at` to itself.  `number`: what the call's
// launches so far have left there, 0 for its first.
uint32_t use(void *at, uint32_t number) {
    auto *word = static_cast<std::atomic<uint32_t> *>(at);
    if (number != 0 && word->load() != number) ++g_failures;
    const uint32_t mine = g_next++;
    word->store(mine);
    if (++g_inside > 1) ++g_side_by_side;
    rest();
    --g_inside;
    if (word->load() != mine) ++g_failures;
    ++g_launches;
    return mine;
}

// Of a call's launches one after the other.
thread_local uint32_t t_last = 0;

}  // namespace

extern "C" {

hipError_t hipGetDevice(int *device) {
    *device = 0;
    return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "?"; }
hipError_t hipDeviceGetAttribute(int *value, hipDeviceAttribute_t, int) {
    *value = 256;
    return hipSuccess;
}
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *status) {
    *status = hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipThreadExchangeStreamCaptureMode(hipStreamCaptureMode *) { return hipSuccess; }
hipError_t hipMalloc(void **p, size_t bytes) {
    *p = std::calloc(1, bytes);  // never freed, as the library's
    return *p != nullptr ? hipSuccess : hipErrorOutOfMemory;
}
hipError_t hipFree(void *p) {
    std::free(p);
    return hipSuccess;
}
hipError_t hipMemsetAsync(void *p, int value, size_t bytes, hipStream_t) {
    std::memset(p, value, bytes);
    return hipSuccess;
}

}  // extern "C"

namespace q4rdna {

int set_error(int code, const char *fmt, ...) {
    std::va_list args;
    va_start(args, fmt);
    std::vprintf(fmt, args);
    va_end(args);
    std::puts("");
    return code;
}

hipError_t launch_append(const AppendArgs &, hipStream_t) { return hipSuccess; }
hipError_t launch_read(const ReadArgs &, hipStream_t) { return hipSuccess; }
hipError_t launch_add_norm(const q4rdna_add_norm_desc &, bool, uint32_t, hipStream_t) { return hipSuccess; }
hipError_t launch_tree(const q4rdna_kv_batch &, const int32_t *, int32_t *, uint64_t *, hipStream_t) { return hipSuccess; }
hipError_t launch_rotate(const RotateArgs &, hipStream_t) { return hipSuccess; }

uint32_t attend_few_rows(uint32_t) { return 8; }
uint64_t attend_many_places(const q4rdna_kv_batch &b, uint32_t group) { return b.tokens * static_cast<uint64_t>(group) / 128 + 1; }
hipError_t launch_attend_few(const AttendArgs &a, uint32_t, uint32_t, hipStream_t) {
    if (a.partials != nullptr) use(a.partials, 0);
    return hipSuccess;
}
hipError_t launch_attend_many(const AttendArgs &a, uint32_t, hipStream_t) {
    if (a.partials != nullptr) use(a.partials, 0);
    return hipSuccess;
}
// The attention's launch and the one that joins its parts.
hipError_t launch_attend_tree(const TreeArgs &a, hipStream_t) {
    if (a.splits == 1) ++g_failures;  // (the call is meant to split)
    use(a.partials, use(a.partials, 0));
    return hipSuccess;
}
hipError_t launch_beam(const BeamArgs &a, hipStream_t) {
    use(a.tops, 0);
    return hipSuccess;
}
hipError_t launch_fork(const ForkArgs &a, uint32_t, uint32_t, hipStream_t) {
    for (uint32_t i = 0; i < 32 * (1 + kForkGates); ++i)
        if (a.arrived[i] != 0) ++g_failures;
    rest();
    return hipSuccess;
}
hipError_t launch_fork_plan(const ForkArgs &a, hipStream_t) {
    t_last = use(a.moves, 0);
    return hipSuccess;
}
hipError_t launch_fork_move(const ForkArgs &a, uint32_t, hipStream_t) {
    t_last = use(a.moves, t_last);
    return hipSuccess;
}

}  // namespace q4rdna

namespace {

alignas(4096) unsigned char g_memory[1 << 16];
void *at(int page) { return g_memory + 256 * page; }

q4rdna_kv_cache a_cache(int i) {
    q4rdna_kv_cache c{};
    c.pages = static_cast<int8_t *>(at(0));
    c.scales = static_cast<float *>(at(1));
    c.open = static_cast<int8_t *>(at(2 + 2 * i));
    c.open_scales = static_cast<float *>(at(3 + 2 * i));
    c.page_count = 100000;
    c.slot_count = 4096;
    c.kv_heads = 8;
    c.head_dim = 128;
    return c;
}

void call(int which, void *stream, uint32_t size) {
    const q4rdna_kv_cache cache = a_cache(0);
    int rc = 0;
    const q4rdna_kv_rows rows{at(0), 1024, 128};
    q4rdna_kv_batch b{};
    b.past = b.cu_tokens = b.table = static_cast<const int32_t *>(at(0));
    b.sequences = 1;
    b.tokens = b.max_tokens = 8;
    b.table_width = 64 * size;
    if (which == 0) {
        q4rdna_kv_tree_desc d{};
        d.q_heads = 32;
        d.q = d.k = d.v = d.out = rows;
        d.seen = static_cast<const uint64_t *>(at(0));
        rc = q4rdna_kv_attend_tree(&cache, &b, &d, stream);
    } else if (which == 1) {
        q4rdna_kv_attend_desc d{};
        d.q_heads = 32;
        d.q = d.out = rows;
        rc = q4rdna_kv_attend(&cache, &b, &d, stream);
    } else if (which == 2) {
        q4rdna_beam_desc d{};
        d.groups = size;
        d.beams = 4;
        d.vocab = 50000;
        d.count = 8;
        d.logits = d.scores = d.out_scores = static_cast<float *>(at(0));
        d.out_rows = d.out_tokens = static_cast<int32_t *>(at(0));
        rc = q4rdna_beam_select(&d, stream);
    } else {
        std::vector<q4rdna_kv_cache> caches;
        for (int i = 0; i < 100; ++i) caches.push_back(a_cache(i));  // more layers than a launch copies
        q4rdna_kv_fork_desc d{};
        d.parents = static_cast<const int32_t *>(at(0));
        d.past = d.table = d.slots = static_cast<int32_t *>(at(0));
        d.sequences = which == 3 ? 500 * size : 4;
        d.table_width = 8;
        d.room = 1;
        rc = q4rdna_kv_fork(caches.data(), which == 3 ? 100 : 2, &d, stream);
    }
    if (rc != Q4RDNA_OK) ++g_failures;
}

}  // namespace

int main() {
    // Four threads on one stream, two on another; sizes grow, so buffers do too.
    std::vector<std::thread> threads;
    for (int t = 0; t < 6; ++t)
        threads.emplace_back([t] {
            for (int i = 0; i < 120; ++i) call((i + t) % 5, at(t < 4 ? 0 : 1), 1 + i / 20);
        });
    for (std::thread &t : threads) t.join();
    std::printf("{\"launches\": %d, \"side_by_side\": %d, \"failures\": %d}\n", g_launches.load(), g_side_by_side.load(), g_failures.load());
    return g_failures != 0;
}
