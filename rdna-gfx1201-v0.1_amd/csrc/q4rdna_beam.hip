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
// Exponentials are fp32's, 16 of a thread's are added up in fp32 and these in 64
// bits.  Of 2^-24 that is 5/2 |x - max| on average, the instruction's 2 and 15
// additions at most, under 2^-18 of the sum; a few 2^-24 as a rule, since they
// differ in sign.  Totals of two beams are off by that, less than the last place of
// fp32 scores of 10 or so, which come in and go out.  (In 64 bits throughout,
// 20 instructions an exponential: 24.5 us rather than 18.0 for 10 each of 5 of 160
// rows of 50257, 12.7 rather than 11.2 for 8 of 4 of 151936, a pass.)
//
// Selection: threads' maxima, several threads' together, 64 or 128 in all; the
// count-th largest of them is a bound that `count` items at least reach, and
// few more.  These go to LDS and each counts how many are before it.  Equal
// logits are told apart by their token, so a bound always cuts; where more items
// reach it than LDS takes, the count-th of those that LDS has is the next bound.
//
// The logits are read once, at far less than a copy's rate: what takes the time
// is one thing after another, load, bound, order, arrival, sums, totals, order.
// 1 of 151936 in fp32 8.0 us, 8 of 4 rows 11.8, 10 of each 5 of 160 rows of 50257
// in bf16 (16 MB) 18.5.
#include "q4rdna_layer_device.h"

namespace q4rdna {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kBeamThreads = 256;
constexpr uint32_t kBeamWaves = kBeamPartials;
constexpr uint32_t kHeld = 1024;  // items that LDS takes

// Bits that order as the numbers do; both zeros are one.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered32(uint32_t u) {
    return __uint_as_float(u ^ (static_cast<uint32_t>(static_cast<int32_t>(~u) >> 31) | 0x80000000u));
}
__device__ __forceinline__ uint64_t ordered(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
    return u ^ (static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double unordered64(uint64_t u) {
    return __builtin_bit_cast(double, u ^ (static_cast<uint64_t>(static_cast<int64_t>(~u) >> 63) | 0x8000000000000000ull));
}

// What is selected, larger first; zero: no item, behind all.
//  Pick    an item of a chunk: ordered logit << 32 | ~token, no two alike.
//  Total   a continuation: by its total, then by row, logit and token.
struct Pick {
    uint64_t key;
    static constexpr bool kPlaced = false;
    __device__ __forceinline__ bool before(const Pick &o) const { return key > o.key; }
};
struct Total {
    uint64_t key, place;
    static constexpr bool kPlaced = true;  // keys may be alike, places not
    __device__ __forceinline__ bool before(const Total &o) const { return key > o.key || (key == o.key && place > o.place); }
};
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane) {
    return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane))) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}
template <int CTRL>
__device__ __forceinline__ uint64_t max_dpp(uint64_t v) {
    const uint64_t o = static_cast<uint64_t>(dpp<CTRL>(static_cast<uint32_t>(v >> 32))) << 32 | dpp<CTRL>(static_cast<uint32_t>(v));
    return o > v ? o : v;
}

template <typename Item>
struct Select {
    Item held[kHeld];
    uint64_t group[128];
    uint32_t ranks[4][128];
    uint32_t count;
    Item chosen;
};

// A key that `count` of the workgroup's threads' largest keys, `mine`, taken
// together by two (count > 32) or four threads, at least reach: the count-th of
// them; 1 where fewer are not zero.
template <typename Item>
__device__ __forceinline__ uint64_t count_th(Select<Item> &s, uint32_t count, uint64_t mine) {
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const bool pairs = count > 32;
    uint64_t g = max_dpp<kDppXor1>(mine);
    if (!pairs) g = max_dpp<kDppXor2>(g);
    if (tid % (pairs ? 2 : 4) == 0) s.group[tid / (pairs ? 2 : 4)] = g;
    __syncthreads();
    // A lane has one or two keys and counts those that are before it, and above
    // these, 2^16 each, those that are not behind it, a quarter in each wave.
    const uint64_t a = s.group[lane], b = pairs ? s.group[lane + 64] : 0;
    uint32_t a_rank = 0, b_rank = 0;
    constexpr uint32_t kLeast = 1u << 16;
#pragma unroll 4
    for (int i = 16 * wave; i < 16 * wave + 16; ++i) {
        const uint64_t o = lane_value(a, i);
        a_rank += o > a ? 1 + kLeast : o == a ? kLeast : 0;
    }
    if (pairs) {
#pragma unroll 1
        for (int i = 16 * wave; i < 16 * wave + 16; ++i) {
            const uint64_t o = lane_value(a, i), p = lane_value(b, i);
            a_rank += p > a ? 1 + kLeast : p == a ? kLeast : 0;
            b_rank += (o > b ? 1 + kLeast : o == b ? kLeast : 0) + (p > b ? 1 + kLeast : p == b ? kLeast : 0);
        }
        s.ranks[wave][lane + 64] = b_rank;
    }
    s.ranks[wave][lane] = a_rank;
    __syncthreads();
    const auto found = [&](uint64_t key, int at) {
        const uint32_t rank = s.ranks[0][at] + s.ranks[1][at] + s.ranks[2][at] + s.ranks[3][at];
        const uint64_t here = __builtin_amdgcn_ballot_w64((rank & 0xffffu) < count && rank >> 16 >= count);
        return here != 0 ? lane_value(key, __builtin_ctzll(here)) : 0;
    };
    uint64_t key = found(a, lane);
    if (pairs && key == 0) key = found(b, lane + 64);
    return key != 0 ? key : 1;
}

// The `count` first of the `n` items in LDS, count <= 128, in order: take(r, item)
// is called once for each place r < count by some thread, with zero where there
// are fewer.
template <typename Item, typename Take>
__device__ __forceinline__ void take_first(const Select<Item> &s, uint32_t n, uint32_t count, Take take) {
    for (uint32_t i = threadIdx.x; i < max(n, count); i += kBeamThreads) {
        if (i >= n) {
            take(i, Item{});
            continue;
        }
        const Item x = s.held[i];
        uint32_t r = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < n; ++j) r += s.held[j].before(x);
        if (r < count) take(r, x);
    }
}
// Whether x reaches the bound.
template <typename Item>
__device__ __forceinline__ bool hold(Select<Item> &s, const Item &bound, const Item &x) {
    if (bound.before(x)) return false;
    const uint32_t at = atomicAdd(&s.count, 1u);
    if (at < kHeld) s.held[at] = x;
    return true;
}
// Sets the count of what is held to zero, between barriers.
template <typename Item>
__device__ __forceinline__ void let_go(Select<Item> &s) {
    __syncthreads();
    if (threadIdx.x == 0) s.count = 0;
    __syncthreads();
}
// The count afterwards, the same for all threads.
template <typename Item>
__device__ __forceinline__ uint32_t held_count(const Select<Item> &s) {
    __syncthreads();
    const uint32_t n = s.count;
    __syncthreads();
    return n;
}
// A thread's share of the first `n` items that are held.
constexpr int kShare = static_cast<int>(kHeld) / kBeamThreads;
template <typename Item>
__device__ __forceinline__ void share_of(const Select<Item> &s, uint32_t n, Item (&share)[kShare]) {
#pragma unroll
    for (int i = 0; i < kShare; ++i) {
        const uint32_t at = threadIdx.x + i * kBeamThreads;
        share[i] = at < n ? s.held[at] : Item{};
    }
}
// Of n <= kHeld items that are held, those that reach a higher bound, `count` at
// least: how many.  By keys, or by places among those with the bound's key.
template <bool PLACES, typename Item>
__device__ __forceinline__ uint32_t tighten(Select<Item> &s, uint32_t count, uint32_t n, Item &bound) {
    Item share[kShare];
    share_of(s, n, share);
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < kShare; ++i) {
        uint64_t at = share[i].key;
        if constexpr (PLACES) at = share[i].key > bound.key ? ~uint64_t{0} : share[i].place;
        mine = max(mine, at);  // (of one type: max() of two would be a double's)
    }
    let_go(s);
    const uint64_t at = count_th(s, count, mine);
    if constexpr (PLACES) bound.place = max(bound.place, at);
    else if (at > bound.key) bound = Item{at};
#pragma unroll
    for (int i = 0; i < kShare; ++i)
        if (share[i].key != 0) hold(s, bound, share[i]);
    return held_count(s);
}
// The same until few are left, or a step leaves out less than a quarter.
__device__ __forceinline__ uint32_t few_of(uint32_t count) { return 2 * count + 64; }
template <typename Item>
__device__ __noinline__ uint32_t shrink(Select<Item> &s, uint32_t count, uint32_t n, Item *bound) {
    Item b = *bound;
    for (bool on = true; on && n > few_of(count);) {
        uint32_t last = n;
        n = tighten<false>(s, count, n, b);
        if constexpr (Item::kPlaced)
            if (4 * n > 3 * last) n = tighten<true>(s, count, last = n, b);
        on = 4 * n <= 3 * last;
    }
    *bound = b;
    return n;
}
// Where more items reach the bound than LDS takes: the count-th of the kHeld that
// are held, which as many of all reach.  Nothing is held afterwards.  (Each time
// all but count of these fall behind, and of others as many as they stand for.)
template <typename Item>
__device__ __noinline__ void raise(Select<Item> &s, uint32_t count, Item *bound) {
    const uint32_t n = shrink(s, count, kHeld, bound);
    for (uint32_t i = threadIdx.x; i < n; i += kBeamThreads) {
        const Item x = s.held[i];
        uint32_t r = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < n; ++j) r += s.held[j].before(x);
        if (r == count - 1) s.chosen = x;
    }
    let_go(s);
    *bound = s.chosen;
}

// The sum over a wave, in every lane.
template <int CTRL>
__device__ __forceinline__ double add_dpp(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return v + __builtin_bit_cast(double, static_cast<uint64_t>(dpp<CTRL>(static_cast<uint32_t>(u >> 32))) << 32 | dpp<CTRL>(static_cast<uint32_t>(u)));
}
__device__ __forceinline__ double wave_sum(double v) {
    v = add_dpp<kDppMirror16>(add_dpp<kDppMirror8>(add_dpp<kDppXor2>(add_dpp<kDppXor1>(v))));
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    double row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) row[i] = __builtin_bit_cast(double, lane_value(u, 16 * i));
    return (row[0] + row[1]) + (row[2] + row[3]);
}
// log x for x > 0 to 2^-39: of x = f 2^e, f in [1/2^.5, 2^.5), by the series of
// 2 atanh((f - 1) / (f + 1)).
__device__ __forceinline__ double log_of(double x) {
    double f = __builtin_amdgcn_frexp_mant(x);
    int e = __builtin_amdgcn_frexp_exp(x);
    if (f < 0.70710678118654752) {
        f += f;
        --e;
    }
    const double s = (f - 1.0) / (f + 1.0), z = s * s;
    double p = 1.0 / 13.0;
    p = fma(p, z, 1.0 / 11.0);
    p = fma(p, z, 1.0 / 9.0);
    p = fma(p, z, 1.0 / 7.0);
    p = fma(p, z, 1.0 / 5.0);
    p = fma(p, z, 1.0 / 3.0);
    p = fma(p, z, 1.0);
    return fma(static_cast<double>(e), 0.69314718055994531, 2.0 * s * p);
}
__device__ __forceinline__ float wave_max(float m) {
    m = fmaxf(m, dpp<kDppXor1>(m));
    m = fmaxf(m, dpp<kDppXor2>(m));
    m = fmaxf(m, dpp<kDppMirror8>(m));
    m = fmaxf(m, dpp<kDppMirror16>(m));
    return max_xor32(max_xor16(m));
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
__device__ __forceinline__ Total total_item(double total, uint32_t beam, uint32_t logit, uint32_t token) {
    static_assert(Q4RDNA_BEAM_MAX_BEAMS == 1 << 8, "beam, logit and token (under 2^24) fill 64 bits");
    return Total{ordered(total), static_cast<uint64_t>(255u - beam) << 56 | static_cast<uint64_t>(logit) << 24 | (~token & 0xffffffu)};
}

// A trip's numbers: a thread has E, in vectors of 16 bytes, at any alignment.
constexpr int E = kBeamTrip / kBeamThreads;
constexpr uint32_t kTrip = kBeamTrip;
template <typename T>
constexpr int V = 16 / static_cast<int>(sizeof(T));
template <typename T>
__device__ __forceinline__ uint32_t token_of(uint32_t base, int e) {
    return base + (e / V<T> * kBeamThreads + threadIdx.x) * V<T> + e % V<T>;
}
// A number of a row; under 2^24 of them, so 32 bits hold the offset.
template <typename V>
__device__ __forceinline__ V row_at(const void *row, uint32_t offset) {
    typedef __attribute__((address_space(1))) const char *gptr_char;
    typedef __attribute__((address_space(1))) const V *gptr;
    return *(gptr)((gptr_char)(uintptr_t)row + offset);
}
// As they lie in memory; -inf behind the row's end.  (They become floats where
// they are used: a conversion here would wait for them.)
template <typename T>
struct Trip {
    typedef T TV __attribute__((ext_vector_type(V<T>), aligned(sizeof(T))));
    TV v[E / V<T>];
};
template <typename T>
__device__ __forceinline__ void load_trip(const T *p, uint32_t base, uint32_t vocab, Trip<T> &x) {
    constexpr uint32_t kSize = sizeof(T);
    if (base + kTrip <= vocab) {
#pragma unroll
        for (int j = 0; j < E / V<T>; ++j) x.v[j] = row_at<typename Trip<T>::TV>(p, kSize * token_of<T>(base, j * V<T>));
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t at = token_of<T>(base, e);
            const T v = row_at<T>(p, kSize * min(at, vocab - 1));
            x.v[e / V<T>][e % V<T>] = at < vocab ? v : static_cast<T>(-__builtin_inff());
        }
    }
}

// Rows in which more logits of a trip reach the bound than LDS takes, as those
// that rise from token to token: the bound becomes the count-th of the trip's and
// of the `before` that were held.
template <typename T>
__device__ __noinline__ void overflown(Select<Pick> &s, const T *p, uint32_t base, uint32_t vocab, uint32_t before, uint32_t count,
                                       Pick *bound) {
    const uint32_t end = min(vocab - base, kTrip);
    const auto trip = [&](auto f) {
        for (uint32_t i = threadIdx.x; i < end; i += kBeamThreads) {
            const float x = static_cast<float>(row_at<T>(p, sizeof(T) * (base + i)));
            if (x == x) f(Pick{static_cast<uint64_t>(ordered(x)) << 32 | static_cast<uint32_t>(~(base + i))});
        }
    };
    Pick share[kShare];
    share_of(s, before, share);
    __syncthreads();
    do {
        raise(s, count, bound);
#pragma unroll
        for (int i = 0; i < kShare; ++i)
            if (share[i].key != 0) hold(s, *bound, share[i]);
        trip([&](const Pick &x) { hold(s, *bound, x); });
    } while (held_count(s) > kHeld);
}

template <typename T>
__global__ __launch_bounds__(kBeamThreads) void beam_kernel(const BeamArgs a) {
    __shared__ union {
        Select<Pick> chunk;
        Select<Total> group;
    } select;
    __shared__ uint32_t ticket;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
    const uint32_t group = row / a.d.beams, beam = row - group * a.d.beams, count = a.d.count;
    const uint32_t lists = a.d.beams * a.chunks;  // of a group
    uint64_t *tops = a.tops + static_cast<size_t>(group) * lists * count;
    uint64_t *stats = a.stats + static_cast<size_t>(group) * lists * kBeamWaves * 2;

    const T *p = static_cast<const T *>(a.d.logits) + group * a.d.group_stride + beam * a.d.beam_stride;
    const uint32_t first = chunk * a.trips * kTrip, trips = min(a.trips, (a.d.vocab - first + kTrip - 1) / kTrip);
    uint64_t *top = tops + static_cast<size_t>(beam) * a.chunks + chunk;
    float m = -__builtin_inff();  // of the thread
    double sum = 0.0;             // of its exponentials, relative to m
    Trip<T> next;
    Select<Pick> &s = select.chunk;
    if (tid == 0) s.count = 0;
    Pick bound = {0};
    uint32_t n = 0;
    for (uint32_t trip = 0; trip <= trips; ++trip) {  // a trip is loaded in the one before
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = static_cast<float>(next.v[e / V<T>][e % V<T>]);
        if (trip < trips) load_trip<T>(p, first + trip * kTrip, a.d.vocab, next);
        if (trip == 0) continue;
        const uint32_t base = first + (trip - 1) * kTrip;
        // (The maximum leaves NaN out; the sum takes it in.)
        float tops_of[E / 8], most = -__builtin_inff();
#pragma unroll
        for (int g = 0; g < E / 8; ++g) {
            tops_of[g] = x[8 * g];
#pragma unroll
            for (int e = 1; e < 8; ++e) tops_of[g] = fmaxf(tops_of[g], x[8 * g + e]);
            most = fmaxf(most, tops_of[g]);
        }
        const float now = fmaxf(m, most), ref = now == -__builtin_inff() ? 0.0f : now;
        float part = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) part += __builtin_amdgcn_exp2f((x[e] - ref) * kLog2e);
        sum = sum * __builtin_amdgcn_exp2f((m - ref) * kLog2e) + part;
        m = now;
        if (trip == 1) {
            int best_at = 0;  // of equal logits the lowest token
#pragma unroll
            for (int e = E - 1; e >= 0; --e) best_at = x[e] == most ? e : best_at;
            bound.key = count_th(s, count, static_cast<uint64_t>(ordered(most)) << 32 | static_cast<uint32_t>(~token_of<T>(base, best_at)));
        }
        const float least = unordered32(max(static_cast<uint32_t>(bound.key >> 32), ordered(-__builtin_inff())));
#pragma unroll
        for (int g = 0; g < E / 8; ++g)
            if (__builtin_amdgcn_ballot_w64(!(tops_of[g] < least)) != 0) {
#pragma unroll
                for (int e = 8 * g; e < 8 * g + 8; ++e)
                    if (x[e] >= least && token_of<T>(base, e) < a.d.vocab) hold(s, bound, Pick{static_cast<uint64_t>(ordered(x[e])) << 32 | static_cast<uint32_t>(~token_of<T>(base, e))});
            }
        const uint32_t before = n;
        n = held_count(s);
        if (n > kHeld) {
            Pick raised = bound;  // (bound itself stays in registers)
            overflown<T>(s, p, base, a.d.vocab, before, count, &raised);
            bound = raised;
            n = held_count(s);
        } else if (n > (trip < trips ? kHeld / 2 : few_of(count))) {
            Pick raised = bound;
            n = shrink(s, count, n, &raised);
            bound = raised;
        }
    }
    take_first(s, n, count, [&](uint32_t r, const Pick &i) {
        const bool there = ~static_cast<uint32_t>(i.key) < a.d.vocab;
        store_agent64(top + static_cast<size_t>(r) * lists, there ? i.key : 0);
    });
    // Each wave's sum by itself.  A NaN, and +inf less itself, have come through it:
    // a maximum of +inf tells them.
    float wave_most = wave_max(m);
    const float wave_ref = wave_most == -__builtin_inff() ? 0.0f : wave_most;
    const double all = wave_sum(sum * __builtin_amdgcn_exp2f((m - wave_ref) * kLog2e));
    if (all != all) wave_most = __builtin_inff();
    if (lane == 0) {
        uint64_t *stat = stats + ((static_cast<size_t>(beam) * a.chunks + chunk) * kBeamWaves + wave) * 2;
        store_agent64(stat, __builtin_bit_cast(uint64_t, all));
        store_agent64(stat + 1, __float_as_uint(wave_most));
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
    // A list to each thread, its first items to the first ones, and so on: the
    // threads' maxima are near each other.  Where these are few a thread they
    // stay in registers, and are under way while the sums are added up.
    const uint32_t width = 1u << (32 - __builtin_clz(max(lists, 2u) - 1));  // of a row of threads
    constexpr int kKept = 4;
    const bool few = width <= kBeamThreads && count <= kKept * (kBeamThreads / width);
    const uint32_t my_list = tid & (width - 1), my_first = tid / width, my_step = kBeamThreads / width;
    uint64_t kept[kKept];
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
        const uint32_t r = my_first + i * my_step;
        kept[i] = few && my_list < lists && r < count ? load_agent64(tops + static_cast<size_t>(r) * lists + my_list) : 0;
    }
    const uint32_t parts = a.chunks * kBeamWaves;
    const auto score_of = [&](uint32_t b) { return a.d.scores == nullptr ? 0.0f : a.d.scores[group * a.d.beams + b]; };
    const auto lse_of = [&](float score, float m, double all) {
        const bool there = __builtin_fabsf(score) < __builtin_inff() && __builtin_fabsf(m) < __builtin_inff();
        return there ? static_cast<double>(m) + log_of(all) : __builtin_nan("");
    };
    const auto load_part = [&](uint32_t b, uint32_t c, double &sum, float &most) {
        const uint64_t *stat = stats + (static_cast<size_t>(b) * parts + min(c, parts - 1)) * 2;
        sum = __builtin_bit_cast(double, load_agent64(stat));
        most = c < parts ? __uint_as_float(static_cast<uint32_t>(load_agent64(stat + 1))) : -__builtin_inff();
    };
    if (parts <= 64) {  // one part a lane, several beams under way together
        constexpr int kBeams = 4;
#pragma unroll 1
        for (uint32_t b0 = wave; b0 < a.d.beams; b0 += 4 * kBeams) {
            float most[kBeams];
            double sum[kBeams];
#pragma unroll
            for (int i = 0; i < kBeams; ++i) load_part(min(b0 + 4 * i, a.d.beams - 1), lane, sum[i], most[i]);
#pragma unroll
            for (int i = 0; i < kBeams; ++i)
                if (b0 + 4 * i < a.d.beams) {
                    const float m = wave_max(most[i]);
                    const double all = wave_sum((most[i] == -__builtin_inff() ? 0.0 : sum[i]) * __builtin_amdgcn_exp2f((most[i] - m) * kLog2e));
                    if (lane == 0) {
                        beam_lse[b0 + 4 * i] = all;
                        beam_score[b0 + 4 * i] = m;
                    }
                }
        }
        // A thread then has a beam: its sum and maximum make way.
        const float score = static_cast<uint32_t>(tid) < a.d.beams ? score_of(tid) : 0.0f;
        __syncthreads();
        if (static_cast<uint32_t>(tid) < a.d.beams) {
            beam_lse[tid] = lse_of(score, beam_score[tid], beam_lse[tid]);
            beam_score[tid] = score;
        }
    } else {
#pragma unroll 1
        for (uint32_t b = wave; b < a.d.beams; b += 4) {
            const float score = score_of(b);
            double sum_of = 0.0;
            float most_of = -__builtin_inff();  // what the lane's parts are relative to
            constexpr int kParts = 4;           // of a lane, under way together
#pragma unroll 1
            for (uint32_t c0 = lane; c0 < parts; c0 += 64 * kParts) {
                float most[kParts], now = most_of;
                double sum[kParts];
#pragma unroll
                for (int i = 0; i < kParts; ++i) load_part(b, c0 + 64 * i, sum[i], most[i]);
#pragma unroll
                for (int i = 0; i < kParts; ++i) now = fmaxf(now, most[i]);
                const float to = now == -__builtin_inff() ? 0.0f : now;
                sum_of *= __builtin_amdgcn_exp2f((most_of - to) * kLog2e);
#pragma unroll
                for (int i = 0; i < kParts; ++i) sum_of += sum[i] * __builtin_amdgcn_exp2f((most[i] - to) * kLog2e);
                most_of = now;
            }
            const float m = wave_max(most_of);
            const double lse = lse_of(score, m, wave_sum(sum_of * __builtin_amdgcn_exp2f((most_of - m) * kLog2e)));
            if (lane == 0) {
                beam_lse[b] = lse;
                beam_score[b] = score;
            }
        }
    }
    __syncthreads();
    // The r-th of a list, of a beam.  A dead beam's items are its first tokens, all
    // at -inf.
    const auto item = [&](uint32_t r, uint32_t list, uint32_t b, uint64_t top) {
        const double lse = beam_lse[b];
        if (lse != lse) return list == b * a.chunks && r < min(count, a.d.vocab) ? total_item(-__builtin_inf(), b, ordered(-__builtin_inff()), r) : Total{0, 0};
        if (top == 0) return Total{0, 0};
        const uint32_t logit = static_cast<uint32_t>(top >> 32);
        return total_item(static_cast<double>(beam_score[b]) + (static_cast<double>(unordered32(logit)) - lse), b, logit, ~static_cast<uint32_t>(top));
    };
    const auto take = [&](uint32_t r, const Total &t) {
        const size_t at = static_cast<size_t>(group) * count + r;
        a.d.out_scores[at] = static_cast<float>(unordered64(t.key));
        a.d.out_rows[at] = static_cast<int32_t>(group * a.d.beams + static_cast<uint32_t>(~t.place >> 56));
        a.d.out_tokens[at] = static_cast<int32_t>(static_cast<uint32_t>(~t.place) & 0xffffffu);
    };
    Select<Total> &g = select.group;
    if (tid == 0) g.count = 0;
    uint64_t best = 0;
    Total least = {0, 0};
    if (few) {
        Total t[kKept];
        const uint32_t my_beam = min(my_list, lists - 1) / a.chunks;
#pragma unroll
        for (int i = 0; i < kKept; ++i) {
            t[i] = Total{0, 0};
            if (i * my_step >= count) continue;
            if (my_list < lists) t[i] = item(my_first + i * my_step, my_list, my_beam, kept[i]);
            best = max(best, t[i].key);
        }
        least.key = count_th(g, count, best);
#pragma unroll
        for (int i = 0; i < kKept; ++i)
            if (i * my_step < count) hold(g, least, t[i]);
    } else {
        // A thread has a block of neighbours of a list, or of several lists.
        // These are sorted: f(t) is called from the first on until it is false.
        const uint32_t across_log2 = min(31 - __builtin_clz(width), 8), across = 1u << across_log2;
        const uint32_t in_block = (count + (kBeamThreads >> across_log2) - 1) >> (8 - across_log2);
        const uint32_t block = (tid >> across_log2) * in_block, block_end = min(block + in_block, count);
        const auto every = [&](auto f) {
#pragma unroll 1
            for (uint32_t list = tid & (across - 1); list < lists; list += across) {
                const uint32_t b = list / a.chunks;
                bool on = true;
#pragma unroll 1
                for (uint32_t r = block; on && r < block_end; r += 4) {
                    uint64_t top[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) top[i] = load_agent64(tops + static_cast<size_t>(min(r + i, block_end - 1)) * lists + list);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (on && r + i < block_end) {
                            const Total t = item(r + i, list, b, top[i]);
                            on = t.key != 0 && f(t);
                        }
                }
            }
        };
        // The blocks' first items bound as above; their last ones stand for a block each.
        uint64_t last = 0;
#pragma unroll 1
        for (uint32_t list = tid & (across - 1); block < count && list < lists; list += across) {
            const uint32_t b = list / a.chunks;
            const uint64_t top = load_agent64(tops + static_cast<size_t>(block) * lists + list);
            const uint64_t end = load_agent64(tops + static_cast<size_t>(block_end - 1) * lists + list);
            best = max(best, item(block, list, b, top).key);
            if (block_end - block == in_block) last = max(last, item(block_end - 1, list, b, end).key);
        }
        least.key = count_th(g, count, best);
        __syncthreads();
        least.key = max(least.key, count_th(g, (count + in_block - 1) / in_block, last));
        every([&](const Total &t) { return hold(g, least, t); });
        while (held_count(g) > kHeld) {
            Total raised = least;
            raise(g, count, &raised);
            least = raised;
            every([&](const Total &t) { return hold(g, least, t); });
        }
    }
    uint32_t found = held_count(g);
    if (found > few_of(count)) {
        Total raised = least;
        found = shrink(g, count, found, &raised);
    }
    take_first(g, found, count, take);
}

}  // namespace

hipError_t launch_beam(const BeamArgs &a, hipStream_t stream) {
    const auto go = [&](auto kernel) { kernel<<<a.d.groups * a.d.beams * a.chunks, kBeamThreads, 0, stream>>>(a); };
    a.d.dtype == Q4RDNA_F32 ? go(beam_kernel<float>) : a.d.dtype == Q4RDNA_F16 ? go(beam_kernel<_Float16>) : go(beam_kernel<__bf16>);
    return hipGetLastError();
}

}  // namespace q4rdna
