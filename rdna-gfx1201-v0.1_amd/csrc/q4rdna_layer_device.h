// Device helpers of the decoder-layer kernels (q4rdna_cache.hip and the others
// that q4rdna_layer.h lists).
#pragma once

#include "q4rdna_device.h"
#include "q4rdna_layer.h"

namespace q4rdna {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// a * b / c.  The usual product fits 32 bits; the 64-bit divisions alone would
// take 0.9 us of a kernel's first steps.
__device__ __forceinline__ uint32_t mul_div(uint32_t a, uint32_t b, uint32_t c) {
    const uint64_t x = static_cast<uint64_t>(a) * b;
    if (x >> 32 == 0) return static_cast<uint32_t>(x) / c;
    return static_cast<uint32_t>(x / c);
}

// 1 / sqrt(x) rounded once, x >= `least`: one step of Newton's iteration on the
// instruction's result (1 ulp), with the exact remainder 1 - x y^2 of two products
// and their errors.  The instruction takes no subnormal x, so where there may be
// one, small ones are scaled by 2^64; zeros, infinities and NaN keep its result.
__device__ __forceinline__ float inverse_root(float x, float least) {
#pragma clang fp contract(off)
    const bool tiny = least < 0x1p-100f && x < 0x1p-100f;
    const float s = tiny ? x * 0x1p64f : x;
    const float y = __builtin_amdgcn_rsqf(s);
    const float t = s * y;
    const float rest = fmaf(-fmaf(s, y, -t), y, fmaf(-t, y, 1.0f));
    constexpr int kPositiveNormal = 0x100;
    const float root = __builtin_amdgcn_classf(s, kPositiveNormal) ? fmaf(0.5f * y, rest, y) : y;
    return tiny ? root * 0x1p32f : root;
}

// 16 bytes of global memory.
__device__ __forceinline__ i32x4 load16(const void *p) { return *(gptr_i32x4)(uintptr_t)p; }
__device__ __forceinline__ void store16(void *p, i32x4 v) { *(gptr_wi32x4)(uintptr_t)p = v; }

// N contiguous elements of type T as floats; `wide`: as vectors of up to 16
// bytes.
template <typename T, int N>
constexpr int kVector = N * sizeof(T) < 16 ? N : 16 / static_cast<int>(sizeof(T));
template <typename T, int N>
__device__ __forceinline__ void load_floats(const T *p, bool wide, float (&x)[N]) {
    constexpr int V = kVector<T, N>;
    typedef T TV __attribute__((ext_vector_type(V)));
    typedef __attribute__((address_space(1))) const TV *gptr_v;
    typedef __attribute__((address_space(1))) const T *gptr_s;
    if (wide) {
#pragma unroll
        for (int i = 0; i < N / V; ++i) {
            const TV v = ((gptr_v)(uintptr_t)p)[i];
#pragma unroll
            for (int e = 0; e < V; ++e) x[V * i + e] = static_cast<float>(v[e]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = static_cast<float>(((gptr_s)(uintptr_t)p)[i]);
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_floats(T *p, bool wide, const float (&x)[N]) {
    constexpr int V = kVector<T, N>;
    typedef T TV __attribute__((ext_vector_type(V)));
    typedef __attribute__((address_space(1))) TV *gptr_v;
    typedef __attribute__((address_space(1))) T *gptr_s;
    if (wide) {
#pragma unroll
        for (int i = 0; i < N / V; ++i) {
            TV v;
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = static_cast<T>(x[V * i + e]);
            ((gptr_v)(uintptr_t)p)[i] = v;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) ((gptr_s)(uintptr_t)p)[i] = static_cast<T>(x[i]);
    }
}

// Reductions over aligned groups of 8 or 16 lanes with DPP moves: quads, then
// the half-row mirror (lane i reads 7 - i), then the row mirror (15 - i); each
// step's partner group already agrees within itself.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __uint_as_float(dpp<CTRL>(__float_as_uint(v)));
}
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E, kDppMirror8 = 0x141, kDppMirror16 = 0x140;
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
    v += dpp<kDppXor1>(v);
    v += dpp<kDppXor2>(v);
    v += dpp<kDppMirror8>(v);
    if (LANES == 16) v += dpp<kDppMirror16>(v);
    return v;
}
template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    v = max(v, dpp<kDppXor1>(v));
    v = max(v, dpp<kDppXor2>(v));
    v = max(v, dpp<kDppMirror8>(v));
    if (LANES == 16) v = max(v, dpp<kDppMirror16>(v));
    return v;
}
// Inclusive sum over the wave's lanes up to this one: shifts within rows of 16
// lanes, then the rows' last lanes into the rows after them.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t scan_step(uint32_t v) {
    return v + static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v = scan_step<0x111, 0xf>(v);
    v = scan_step<0x112, 0xf>(v);
    v = scan_step<0x114, 0xf>(v);
    v = scan_step<0x118, 0xf>(v);
    v = scan_step<0x142, 0xa>(v);
    return scan_step<0x143, 0xc>(v);
}
__device__ __forceinline__ float max_xor16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_xor32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Keeps the scheduler from moving instructions across: it would issue the
// loads or products of many tiles ahead and run out of registers.
__device__ __forceinline__ void tile_end() { __builtin_amdgcn_sched_barrier(0); }

// Two floats at once, device scope (see load_agent).
__device__ __forceinline__ f32x2 load_agent2(const float *p) {
    typedef __attribute__((address_space(1))) const uint64_t *gptr_cu64;
    const uint64_t v = __hip_atomic_load((gptr_cu64)(uintptr_t)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return __builtin_bit_cast(f32x2, v);
}

__device__ __forceinline__ void count_fault(const q4rdna_kv_cache &c) {
    if (c.faults != nullptr) atomicAdd(c.faults, 1u);
}

// One sequence of a step.
struct Seq {
    int first;   // its first token in the step
    int count;   // its tokens in the step
    int past;    // its tokens in the cache before them
    int length;  // past + count
    int slot;
    bool ok;     // every entry is in range
};
__device__ __forceinline__ Seq seq_of(const q4rdna_kv_batch &b, const q4rdna_kv_cache &c, uint32_t i) {
    Seq s;
    s.first = b.cu_tokens ? b.cu_tokens[i] : static_cast<int>(i);
    const int end = b.cu_tokens ? b.cu_tokens[i + 1] : static_cast<int>(i) + 1;
    s.past = b.past[i];
    s.slot = b.slots ? b.slots[i] : static_cast<int>(i);
    s.ok = s.first >= 0 && end >= s.first && static_cast<uint32_t>(end) <= b.tokens;
    s.count = s.ok ? end - s.first : 0;
    const int64_t room = static_cast<int64_t>(b.table_width) * kKvBlock;  // at most 2^30
    s.ok = s.ok && static_cast<uint32_t>(s.count) <= b.max_tokens && s.past >= 0 &&
           static_cast<int64_t>(s.past) + s.count <= room && static_cast<uint32_t>(s.slot) < c.slot_count;
    s.length = s.ok ? s.past + s.count : 0;
    return s;
}

// The last i in [0, n) with key(i) <= x, for ascending keys (0 if none): 64
// keys a trip, a lane each.
template <typename F>
__device__ __forceinline__ uint32_t last_not_past(uint32_t n, int64_t x, F key) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0;
    for (uint32_t step = n > 4096 ? 4096 : n > 64 ? 64 : 1;; step >>= 6) {
        // lanes look at lo, lo + step, ...; the last that fits is the next lo
        const uint32_t i = lo + lane * step;
        const uint64_t fits = __builtin_amdgcn_ballot_w64(i < n && key(i) <= x);
        // ascending keys give a run of ones; anything else still gives an index in range
        lo += fits == 0 ? 0 : (63 - __builtin_clzll(fits)) * step;
        if (step == 1) return lo;
    }
}

// The sequence that owns `place` (kv_places): the last one whose first place
// is not past it.  To be called by whole waves.
__device__ __forceinline__ uint32_t place_seq(const q4rdna_kv_batch &b, uint32_t place, uint32_t *first_place) {
    if (b.cu_tokens == nullptr) {
        *first_place = place;
        return place;
    }
    auto key = [&](uint32_t i) { return static_cast<int64_t>(b.cu_tokens[i]) / kKvBlock + 2ll * i; };
    const uint32_t i = __builtin_amdgcn_readfirstlane(last_not_past(b.sequences, place, key));
    const int64_t base = key(i);
    *first_place = base < 0 || base > place ? place : static_cast<uint32_t>(base);
    return i;
}

// The sequence of token n of the step: the last one that starts at or before
// it.  To be called by whole waves, n the same in all lanes.
__device__ __forceinline__ uint32_t wave_token_seq(const q4rdna_kv_batch &b, uint32_t n) {
    if (b.cu_tokens == nullptr) return n;
    return __builtin_amdgcn_readfirstlane(
        last_not_past(b.sequences, n, [&](uint32_t i) { return static_cast<int64_t>(b.cu_tokens[i]); }));
}
// The same for each lane by itself.
__device__ __forceinline__ uint32_t token_seq(const q4rdna_kv_batch &b, uint32_t n) {
    if (b.cu_tokens == nullptr) return n;
    uint32_t lo = 0, hi = b.sequences;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (b.cu_tokens[mid] <= static_cast<int64_t>(n))
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

__device__ __forceinline__ size_t page_tile(const q4rdna_kv_cache &c, int page, uint32_t head) {
    return (static_cast<size_t>(page) * c.kv_heads + head) * 2u * kKvBlock * c.head_dim;
}
// The open block of parity block & 1 of a slot: offset of its four planes of a
// head, and of its two rows of token scales.
__device__ __forceinline__ size_t open_tile(const q4rdna_kv_cache &c, int slot, int block, uint32_t head) {
    return ((static_cast<size_t>(slot) * 2 + (block & 1)) * c.kv_heads + head) * 4u * kKvBlock * c.head_dim;
}
__device__ __forceinline__ size_t open_scale_row(const q4rdna_kv_cache &c, int slot, int block, uint32_t head) {
    return ((static_cast<size_t>(slot) * 2 + (block & 1)) * c.kv_heads + head) * 2u * kKvBlock;
}

}  // namespace q4rdna
