// Beam search's selection (q4rdna_beam_select): log-softmax of rows of logits,
// the beams' scores, and the largest totals of each group.
//
// One launch.  A workgroup takes a chunk of one row into registers, reads it
// once, and leaves the chunk's maximum, its sum of exponentials and its `count`
// largest logits; a total rises with its row's logit, so a group's best are
// among these.  The last workgroup of a group to arrive adds up the rows' sums
// in the chunks' order, makes the totals in 64 bits and selects again: the
// results do not depend on the order of arrival.
//
// Selection: threads' maxima, several threads' together, 64 or 128 in all; the
// count-th largest of them is a bound that `count` items at least reach, and
// few more.  These go to LDS and each counts how many are before it.  Equal
// items are told apart by their place, so a bound always cuts; where more items
// reach it than LDS takes, as in rows that are sorted, the bound is raised by
// halving.
#include "q4rdna_layer_device.h"

namespace q4rdna {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kBeamThreads = 256;
constexpr uint32_t kHeld = 1024;  // items that LDS takes

// Bits that order as the numbers do; both zeros are one.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) {
    return __uint_as_float(u ^ (static_cast<uint32_t>(static_cast<int32_t>(~u) >> 31) | 0x80000000u));
}
__device__ __forceinline__ uint64_t ordered(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
    return u ^ (static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double unordered(uint64_t u) {
    return __builtin_bit_cast(double, u ^ (static_cast<uint64_t>(static_cast<int64_t>(~u) >> 63) | 0x8000000000000000ull));
}

// What is selected: by `rank`, equal ones by `place`, larger first.  {0, 0}: no
// item, behind all.
struct Item {
    uint64_t rank, place;
};
__device__ __forceinline__ bool before(const Item &a, const Item &b) {
    return a.rank > b.rank || (a.rank == b.rank && a.place > b.place);
}
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane) {
    return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane))) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}
template <int CTRL>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
    return static_cast<uint64_t>(dpp<CTRL>(static_cast<uint32_t>(v >> 32))) << 32 | dpp<CTRL>(static_cast<uint32_t>(v));
}
template <int CTRL>
__device__ __forceinline__ Item best_dpp(const Item &a) {
    const Item b = {dpp64<CTRL>(a.rank), dpp64<CTRL>(a.place)};
    return before(b, a) ? b : a;
}

struct Select {
    Item held[kHeld];
    Item group[128];
    uint32_t count;
};

// The `count` first items, count <= 128, in order: take(r, item) is called once
// for each place r < count by some thread, with {0, 0} where there are fewer
// items.  `mine` is the first of the thread's items, each(f) calls f with all of
// them.  Every thread of the workgroup calls it.
template <typename Each, typename Take>
__device__ __forceinline__ void select_first(Select &s, uint32_t count, const Item &mine, Each each, Take take) {
    const int tid = threadIdx.x, lane = tid & 63;
    const bool pairs = count > 64;  // 128 groups of two threads, else 64 of four
    Item g = best_dpp<kDppXor1>(mine);
    if (!pairs) g = best_dpp<kDppXor2>(g);
    if (tid % (pairs ? 2 : 4) == 0) s.group[tid / (pairs ? 2 : 4)] = g;
    if (tid == 0) s.count = 0;
    __syncthreads();
    // Each wave finds the count-th group by itself: a lane has one or two and
    // counts those before it.
    Item bound;
    {
        const Item a = s.group[lane];
        uint32_t a_rank = 0;
        if (!pairs) {
            for (int i = 0; i < 64; ++i) {
                const Item o = {lane_value(a.rank, i), lane_value(a.place, i)};
                a_rank += before(o, a) || (i < lane && o.rank == a.rank && o.place == a.place);
            }
            const uint64_t at = __builtin_amdgcn_ballot_w64(a_rank == count - 1);
            const int owner = __builtin_ctzll(at | 1ull << 63);
            bound = {lane_value(a.rank, owner), lane_value(a.place, owner)};
        } else {
            const Item b = s.group[lane + 64];
            uint32_t b_rank = 0;
            for (int i = 0; i < 64; ++i) {
                const Item o = {lane_value(a.rank, i), lane_value(a.place, i)}, p = {lane_value(b.rank, i), lane_value(b.place, i)};
                a_rank += before(o, a) || (i < lane && o.rank == a.rank && o.place == a.place);
                a_rank += before(p, a);
                b_rank += before(o, b) || (o.rank == b.rank && o.place == b.place);
                b_rank += before(p, b) || (i < lane && p.rank == b.rank && p.place == b.place);
            }
            const uint64_t at = __builtin_amdgcn_ballot_w64(a_rank == count - 1), bt = __builtin_amdgcn_ballot_w64(b_rank == count - 1);
            const int owner = __builtin_ctzll((at != 0 ? at : bt) | 1ull << 63);
            bound = at != 0 ? Item{lane_value(a.rank, owner), lane_value(a.place, owner)}
                            : Item{lane_value(b.rank, owner), lane_value(b.place, owner)};
        }
    }
    if (bound.rank == 0) bound = {1, 0};  // fewer groups with items than `count`: all items
    // How many reach a bound.
    const auto reach = [&](const Item &at) {
        uint32_t n = 0;
        each([&](const Item &x) { n += !before(at, x); });
        if (n != 0) atomicAdd(&s.count, n);
        __syncthreads();
        const uint32_t all = s.count;
        __syncthreads();
        if (tid == 0) s.count = 0;
        __syncthreads();
        return all;
    };
    uint32_t n = reach(bound);
    if (n > kHeld) {
        // The largest rank that `count` items at least reach, then the same of the places: the
        // bound is then the count-th item itself.
        Item low = {bound.rank, 0}, high = {~0ull, 0};  // low is reached by enough, high is not
        while (high.rank - low.rank > 1) {
            const Item mid = {low.rank + (high.rank - low.rank) / 2, 0};
            (reach(mid) >= count ? low : high) = mid;
        }
        high = {low.rank, ~0ull};
        while (high.place - low.place > 1) {
            const Item mid = {low.rank, low.place + (high.place - low.place) / 2};
            (reach(mid) >= count ? low : high) = mid;
        }
        bound = low;
    }
    each([&](const Item &x) {
        if (!before(bound, x)) s.held[atomicAdd(&s.count, 1u)] = x;
    });
    __syncthreads();
    n = s.count;
    for (uint32_t i = tid; i < max(n, count); i += kBeamThreads) {
        if (i >= n) {
            take(i, Item{0, 0});
            continue;
        }
        const Item x = s.held[i];
        uint32_t r = 0;
        for (uint32_t j = 0; j < n; ++j) r += before(s.held[j], x);
        if (r < count) take(r, x);
    }
    __syncthreads();
}

// What a chunk leaves: its items' logits (ordered) and tokens in `top`, and
// max and sum; max NaN: the row has a NaN or +inf.
struct ChunkStat {
    double sum;  // of exp(logit - max)
    float max;
    uint32_t unused;
};

// N numbers of a row, of any alignment.
template <typename T, int N>
__device__ __forceinline__ void load_any(const T *p, float (&x)[N]) {
    typedef T TV __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    typedef __attribute__((address_space(1))) const TV *gptr;
    const TV v = *(gptr)(uintptr_t)p;
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = static_cast<float>(v[e]);
}

__device__ __forceinline__ uint64_t load_agent64(const uint64_t *p) {
    typedef __attribute__((address_space(1))) const uint64_t *gptr_cu64;
    return __hip_atomic_load((gptr_cu64)(uintptr_t)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_agent64(uint64_t *p, uint64_t v) {
    __hip_atomic_store((gptr_au64)(uintptr_t)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A continuation: by its total, then by its row (lower first), its logit and its
// token (lower first).
__device__ __forceinline__ Item total_item(double total, uint32_t beam, uint32_t logit, uint32_t token) {
    static_assert(Q4RDNA_BEAM_MAX_BEAMS == 1 << 8, "beam, logit and token (under 2^24) fill 64 bits");
    return Item{ordered(total), static_cast<uint64_t>(255u - beam) << 56 | static_cast<uint64_t>(logit) << 24 | (~token & 0xffffffu)};
}

__device__ __forceinline__ bool alive(const q4rdna_beam_desc &d, uint32_t row) {
    return d.scores == nullptr || __builtin_fabsf(d.scores[row]) < __builtin_inff();
}

template <int E, typename T>
__global__ __launch_bounds__(kBeamThreads) void beam_kernel(const BeamArgs a) {
    constexpr int V = E * sizeof(T) < 16 ? E : 16 / static_cast<int>(sizeof(T));
    __shared__ Select select;
    __shared__ float wave_max[4];
    __shared__ double wave_sum[4];
    __shared__ uint32_t ticket;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
    const uint32_t group = row / a.d.beams, beam = row - group * a.d.beams, count = a.d.count;
    const uint32_t lists = a.d.beams * a.chunks;  // of a group
    uint64_t *tops = a.tops + static_cast<size_t>(group) * lists * count;
    uint64_t *stats = a.stats + static_cast<size_t>(group) * lists * 2;

    if (alive(a.d, row)) {
        const T *p = static_cast<const T *>(a.d.logits) + group * a.d.group_stride + beam * a.d.beam_stride;
        const uint32_t first = chunk * (kBeamThreads * E);
        float x[E];
        uint32_t valid = 0;  // bits of the thread's vectors' elements that are there
#pragma unroll
        for (int j = 0; j < E / V; ++j) {
            const uint32_t at = first + (j * kBeamThreads + tid) * V;
            float v[V];
            if (at + V <= a.d.vocab) {
                load_any<T, V>(p + at, v);
                valid |= ((1u << V) - 1u) << (V * j);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    v[e] = 0.0f;
                    if (at + e < a.d.vocab) {
                        v[e] = static_cast<float>(p[at + e]);
                        valid |= 1u << (V * j + e);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < V; ++e) x[V * j + e] = v[e];
        }
        // The maximum, with NaN and +inf as +inf.
        float most = -__builtin_inff();
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (!(x[e] < __builtin_inff())) x[e] = __builtin_inff();
            if (valid >> e & 1) most = fmaxf(most, x[e]);
        }
        // The thread's first item: of equal logits the lowest token.
        Item mine = {0, 0};
#pragma unroll
        for (int e = E - 1; e >= 0; --e)
            if ((valid >> e & 1) && x[e] == most)
                mine = {static_cast<uint64_t>(ordered(x[e])), static_cast<uint64_t>(~(first + (e / V * kBeamThreads + tid) * V + e % V))};
        float m = most;
        m = fmaxf(m, dpp<kDppXor1>(m));
        m = fmaxf(m, dpp<kDppXor2>(m));
        m = fmaxf(m, dpp<kDppMirror8>(m));
        m = fmaxf(m, dpp<kDppMirror16>(m));
        m = max_xor32(max_xor16(m));
        if (lane == 0) wave_max[wave] = m;
        __syncthreads();
        m = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
        // Up to 32 exponentials in 32 bits, all sums of them in 64.
        const float ref = m == -__builtin_inff() ? 0.0f : m;
        float part = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (valid >> e & 1) part += __builtin_amdgcn_exp2f((x[e] - ref) * kLog2e);
        double sum = part;
#pragma unroll
        for (int s = 32; s != 0; s >>= 1) sum += __shfl_xor(sum, s);
        if (lane == 0) wave_sum[wave] = sum;
        uint64_t *top = tops + static_cast<size_t>(beam) * a.chunks + chunk;
        select_first(select, count, mine,
                     [&](auto f) {
#pragma unroll
                         for (int e = 0; e < E; ++e)
                             if (valid >> e & 1)
                                 f(Item{static_cast<uint64_t>(ordered(x[e])),
                                        static_cast<uint64_t>(~(first + (e / V * kBeamThreads + tid) * V + e % V))});
                     },
                     [&](uint32_t r, const Item &i) { store_agent64(top + static_cast<size_t>(r) * lists, i.rank << 32 | static_cast<uint32_t>(i.place)); });
        if (tid == 0) {
            uint64_t *stat = stats + (static_cast<size_t>(beam) * a.chunks + chunk) * 2;
            store_agent64(stat, __builtin_bit_cast(uint64_t, (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3])));
            store_agent64(stat + 1, __float_as_uint(m));
        }
    }

    // The group's last workgroup goes on.
    wait_stores();
    __syncthreads();
    if (tid == 0) ticket = add_agent(a.arrived + group, 1u);
    __syncthreads();
    if (ticket != lists - 1) return;
    if (tid == 0) store_agent(a.arrived + group, 0u);
    // A beam's log-sum-exp, NaN where it has no continuation, and its score.
    __shared__ double beam_lse[Q4RDNA_BEAM_MAX_BEAMS];
    __shared__ float beam_score[Q4RDNA_BEAM_MAX_BEAMS];
    for (uint32_t b = wave; b < a.d.beams; b += 4) {
        const uint32_t r = group * a.d.beams + b;
        double lse = __builtin_nan("");
        if (alive(a.d, r)) {
            float m = -__builtin_inff();
            for (uint32_t c = lane; c < a.chunks; c += 64)
                m = fmaxf(m, __uint_as_float(static_cast<uint32_t>(load_agent64(stats + (static_cast<size_t>(b) * a.chunks + c) * 2 + 1))));
            m = fmaxf(m, dpp<kDppXor1>(m));
            m = fmaxf(m, dpp<kDppXor2>(m));
            m = fmaxf(m, dpp<kDppMirror8>(m));
            m = fmaxf(m, dpp<kDppMirror16>(m));
            m = max_xor32(max_xor16(m));
            double sum = 0.0;
            if (__builtin_fabsf(m) < __builtin_inff()) {
                for (uint32_t c = lane; c < a.chunks; c += 64) {
                    const uint64_t *stat = stats + (static_cast<size_t>(b) * a.chunks + c) * 2;
                    const float cm = __uint_as_float(static_cast<uint32_t>(load_agent64(stat + 1)));
                    const double cs = __builtin_bit_cast(double, load_agent64(stat));
                    if (cm > -__builtin_inff()) sum += cs * exp(static_cast<double>(cm) - static_cast<double>(m));
                }
#pragma unroll
                for (int s = 32; s != 0; s >>= 1) sum += __shfl_xor(sum, s);
                lse = static_cast<double>(m) + log(sum);
            }
        }
        if (lane == 0) {
            beam_lse[b] = lse;
            beam_score[b] = a.d.scores == nullptr ? 0.0f : a.d.scores[r];
        }
    }
    __syncthreads();
    // The lists' first items, then their second ones, and so on: the threads'
    // maxima are near each other.  A dead beam's items are its first tokens, all
    // at -inf.
    const auto item = [&](uint32_t r, uint32_t list) {
        const uint32_t b = list / a.chunks;
        const double lse = beam_lse[b];
        if (lse != lse) return list == b * a.chunks && r < a.d.vocab ? total_item(-__builtin_inf(), b, ordered(-__builtin_inff()), r) : Item{0, 0};
        const uint64_t top = load_agent64(tops + static_cast<size_t>(r) * lists + list);
        if (top == 0) return Item{0, 0};
        const uint32_t logit = static_cast<uint32_t>(top >> 32);
        return total_item(static_cast<double>(beam_score[b]) + (static_cast<double>(unordered(logit)) - lse), b, logit, ~static_cast<uint32_t>(top));
    };
    const auto each = [&](auto f) {
        for (uint32_t i = tid; i < lists * count; i += kBeamThreads) {
            const uint32_t r = i / lists;
            const Item x = item(r, i - r * lists);
            if (x.rank != 0) f(x);
        }
    };
    Item mine = {0, 0};
    each([&](const Item &x) {
        if (before(x, mine)) mine = x;
    });
    select_first(select, count, mine, each, [&](uint32_t r, const Item &i) {
        const size_t at = static_cast<size_t>(group) * count + r;
        a.d.out_scores[at] = static_cast<float>(unordered(i.rank));
        a.d.out_rows[at] = static_cast<int32_t>(group * a.d.beams + static_cast<uint32_t>(~i.place >> 56));
        a.d.out_tokens[at] = static_cast<int32_t>(static_cast<uint32_t>(~i.place) & 0xffffffu);
    });
}

}  // namespace

template <int E>
static void launch_beam_as(const BeamArgs &a, hipStream_t stream) {
    const auto go = [&](auto kernel) { kernel<<<a.d.groups * a.d.beams * a.chunks, kBeamThreads, 0, stream>>>(a); };
    a.d.dtype == Q4RDNA_F32 ? go(beam_kernel<E, float>) : a.d.dtype == Q4RDNA_F16 ? go(beam_kernel<E, _Float16>) : go(beam_kernel<E, __bf16>);
}
hipError_t launch_beam(const BeamArgs &a, hipStream_t stream) {
    switch (a.each) {
        case 4: launch_beam_as<4>(a, stream); break;
        case 8: launch_beam_as<8>(a, stream); break;
        case 16: launch_beam_as<16>(a, stream); break;
        default: launch_beam_as<32>(a, stream); break;
    }
    return hipGetLastError();
}

}  // namespace q4rdna
