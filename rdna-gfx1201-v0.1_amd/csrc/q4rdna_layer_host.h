// What the decoder-layer entry points share (q4rdna_layer.cpp,
// q4rdna_branch.cpp): argument checks, the device that a call runs on, scratch.
#pragma once

#include <atomic>
#include <exception>
#include <mutex>

#include "q4rdna_layer.h"
#include "q4rdna_runtime.h"

namespace q4rdna {

inline bool aligned(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

inline uint32_t size_of(uint32_t dtype) { return dtype == Q4RDNA_F32 ? 4 : 2; }

// No exception leaves a C entry point.
template <typename F>
int guarded(F body) {
    try {
        return body();
    } catch (const std::exception &e) {
        return set_error(Q4RDNA_ERR_MEMORY, "%s", e.what());
    }
}

inline int launched(hipError_t e, const char *what) {
    return e == hipSuccess ? Q4RDNA_OK : set_error(Q4RDNA_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

// A call runs on the cache's device, whatever the calling thread's current one,
// which it gets back.
class OnDevice {
public:
    explicit OnDevice(int device) {
        if (hipGetDevice(&saved_) != hipSuccess) saved_ = -1;
        if (saved_ == device) return;
        switched_ = hipSetDevice(device) == hipSuccess;
        if (!switched_) {
            (void)hipGetLastError();
            status_ = set_error(Q4RDNA_ERR_ARGUMENT, "the cache lives on device %d, which cannot be used", device);
        }
    }
    ~OnDevice() {
        if (switched_ && saved_ >= 0) (void)hipSetDevice(saved_);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
    int status() const { return status_; }

private:
    int saved_ = -1, status_ = Q4RDNA_OK;
    bool switched_ = false;
};

// HIP launches fewer than 2^32 threads.
constexpr uint64_t most_workgroups(uint32_t threads) { return 0xffffffffu / threads; }

// Compute units of a device, looked up once.
inline uint32_t cu_count(int device) {
    static std::atomic<uint32_t> g_cus[64];
    if (device < 0 || device >= 64) return 256;
    uint32_t n = g_cus[device].load(std::memory_order_relaxed);
    if (n != 0) return n;
    int v = 0;
    if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || v <= 0) {
        (void)hipGetLastError();
        return 256;
    }
    g_cus[device].store(static_cast<uint32_t>(v), std::memory_order_relaxed);
    return static_cast<uint32_t>(v);
}

// Checks that need no device come first, so a malformed call is refused the
// same way with and without one.
inline int check_cache(const q4rdna_kv_cache *c) {
    if (c == nullptr || c->pages == nullptr || c->scales == nullptr || c->open == nullptr || c->open_scales == nullptr)
        return set_error(Q4RDNA_ERR_ARGUMENT, "null cache or cache buffer");
    if (c->head_dim != 64 && c->head_dim != 128)
        return set_error(Q4RDNA_ERR_ARGUMENT, "head_dim is %u: 64 and 128 are supported", c->head_dim);
    if (c->kv_heads == 0 || c->kv_heads > 1024 || c->page_count == 0 || c->page_count > 0x7fffffffu || c->slot_count == 0 ||
        c->slot_count > 0x7fffffffu)
        return set_error(Q4RDNA_ERR_ARGUMENT, "cache of %u pages, %u slots, %u kv heads", c->page_count, c->slot_count,
                         c->kv_heads);
    if (!aligned(c->pages, 16) || !aligned(c->scales, 8) || !aligned(c->open, 16) || !aligned(c->open_scales, 16) ||
        !aligned(c->faults, 4))
        return set_error(Q4RDNA_ERR_ARGUMENT, "misaligned cache buffer");
    return Q4RDNA_OK;
}

inline int check_batch(const q4rdna_kv_batch *b) {
    if (b == nullptr) return set_error(Q4RDNA_ERR_ARGUMENT, "null batch");
    if (b->sequences == 0 || b->tokens == 0) return Q4RDNA_OK;  // nothing to do
    if (b->past == nullptr || b->table == nullptr) return set_error(Q4RDNA_ERR_ARGUMENT, "null past or table");
    if (!aligned(b->past, 4) || !aligned(b->cu_tokens, 4) || !aligned(b->table, 4) || !aligned(b->slots, 4))
        return set_error(Q4RDNA_ERR_ARGUMENT, "misaligned batch array");
    if (b->sequences > 65535 || b->tokens > 0x3fffffffu || b->table_width == 0 || b->table_width > (1u << 24))
        return set_error(Q4RDNA_ERR_ARGUMENT, "step of %u sequences, %u tokens, %u table columns", b->sequences, b->tokens,
                         b->table_width);
    if (b->max_tokens == 0 || (b->cu_tokens == nullptr && (b->tokens != b->sequences || b->max_tokens != 1)))
        return set_error(Q4RDNA_ERR_ARGUMENT, "%u tokens of %u sequences, at most %u each: without cu_tokens each has one",
                         b->tokens, b->sequences, b->max_tokens);
    return Q4RDNA_OK;
}

inline int check_rows(const q4rdna_kv_rows &r, uint32_t dtype, const char *name) {
    if (r.data == nullptr) return set_error(Q4RDNA_ERR_ARGUMENT, "null %s", name);
    if (!aligned(r.data, size_of(dtype))) return set_error(Q4RDNA_ERR_ARGUMENT, "misaligned %s", name);
    return Q4RDNA_OK;
}

inline int check_dtype(uint32_t dtype) {
    return dtype > Q4RDNA_BF16 ? set_error(Q4RDNA_ERR_ARGUMENT, "unknown dtype %u", dtype) : Q4RDNA_OK;
}

inline int check_heads(uint32_t q_heads, uint32_t kv_heads) {
    if (q_heads == 0 || q_heads % kv_heads != 0 || q_heads > 32768)
        return set_error(Q4RDNA_ERR_ARGUMENT, "%u query heads over %u kv heads", q_heads, kv_heads);
    return Q4RDNA_OK;
}

// Whether every row starts at a multiple of `elements`.
inline bool wide_rows(const q4rdna_kv_rows &r, uint32_t dtype, int64_t elements) {
    return aligned(r.data, elements * size_of(dtype)) && r.token_stride % elements == 0 && r.head_stride % elements == 0;
}

// Attention's partial results and arrival counters per (device, stream), under
// the same rules as the GEMVs' exchange slots (q4rdna_runtime.cpp): outgrown
// buffers are kept, since launches still queued and captured graphs use them,
// and nothing is allocated while the stream is being captured.  All calls of a
// stream share them, and some leave in one launch what the next one reads: a call
// holds them from here to its last launch, so that no other thread's launch on
// the stream comes between.
struct Scratch {
    float *partials = nullptr;
    uint32_t *arrived = nullptr;
    std::unique_lock<std::mutex> held;
};
int get_scratch(int device, hipStream_t stream, size_t floats, size_t jobs, Scratch *out);

}  // namespace q4rdna
