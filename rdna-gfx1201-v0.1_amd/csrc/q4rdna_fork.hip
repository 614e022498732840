// Sequences that go on from others (q4rdna_kv_fork).
//
// What is decided: each sequence's parent, length and slot, which open blocks are
// copied, and which pages are free, in the order in which they are given out.
// What takes the time is copying the open blocks.
//
// fork_kernel, for up to 256 sequences and tables of up to 2^15 entries, does all
// in one launch.  For larger ones fork_plan_kernel, one workgroup, decides, and
// fork_move_kernel carries it out: a workgroup renames some columns of the table,
// all rows of which it has read before it writes the first, and others copy.
//
// Measured, with the plan in a launch of its own and in one launch: 4 sequences
// of 700 tokens, 4 layers of 8 heads by 128 5.6 + 4.4 and 6.6 us; 8 of 4001, 36
// layers (153 MB read and written) 6.5 + 29.7 and 30.1, a large copy's rate; 200
// of 10 .. 8000, 12 layers of 4 by 64 (212 MB) 11.4 + 42.5 and 48.5.
#include "q4rdna_layer_device.h"

namespace q4rdna {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kBlock = static_cast<int>(kKvBlock);

// Sum of v over the threads before this one; `all` receives that of all.
template <int THREADS>
__device__ __forceinline__ uint32_t threads_before(uint32_t v, uint32_t *totals, uint32_t *all) {
    const int lane = threadIdx.x & 63, wave = wave_id();
    const uint32_t upto = wave_scan(v);
    __syncthreads();  // the totals of the call before have been read
    if (lane == 63) totals[wave] = upto;
    __syncthreads();
    uint32_t before = 0, sum = 0;
    for (int w = 0; w < THREADS / 64; ++w) {
        const uint32_t t = totals[w];
        before += w < wave ? t : 0;
        sum += t;
    }
    *all = sum;
    return before + upto - v;
}

// The open block, where it holds tokens, and those that the next `room` tokens
// behind `past` touch: from past / 64 up to this one.
__device__ __forceinline__ int room_end(const q4rdna_kv_fork_desc &d, int past) {
    const uint64_t end = (static_cast<uint64_t>(past) + d.room + kBlock - 1) / kBlock;
    return static_cast<int>(min(end, static_cast<uint64_t>(d.table_width)));
}

// Four entries of a row, at any of them.
__device__ __forceinline__ i32x4 load_entries(const int32_t *p) {
    typedef int32_t Four __attribute__((ext_vector_type(4), aligned(4)));
    return *(__attribute__((address_space(1))) const Four *)(uintptr_t)p;
}

// Sets the bits of the pages of full blocks, `longest` in a row at most, and of
// those that are kept.
template <int THREADS>
__device__ __forceinline__ void mark_pages(const ForkArgs &a, uint32_t longest, const int32_t *parent, const int32_t *past,
                                           const int32_t *first, uint32_t *used) {
    const int tid = threadIdx.x, n = static_cast<int>(a.d.sequences), width = static_cast<int>(a.d.table_width);
    // Each parent's entries once: four entries of a thread, kEach
    // times in flight, 2^log2 threads a row.
    constexpr int kEach = 4;
    const int log2 = longest <= 4 ? 0 : 32 - __builtin_clz((longest - 1) / 4);
    const uint64_t units = longest == 0 ? 0 : static_cast<uint64_t>(n) << log2;
    for (uint64_t u0 = tid; u0 < units; u0 += kEach * THREADS) {
        i32x4 page[kEach];
        int have[kEach];
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            const uint64_t u = u0 + static_cast<uint64_t>(x) * THREADS;
            const int i = min(static_cast<int>(u >> log2), n - 1), b = 4 * static_cast<int>(u & ((1ull << log2) - 1));
            const int p = parent[i], full = past[i] / kBlock;
            have[x] = 0;
            if (u < units && b < full && first[p] == i) {
                const int at = max(min(b, width - 4), 0);  // within the row, some entries twice
                const int32_t *row = a.d.table + static_cast<size_t>(p) * width + at;
                have[x] = full - at;
                if (width >= 4) page[x] = load_entries(row);
                else page[x] = i32x4{row[0], row[width / 2], row[width - 1], 0};  // all of up to three
            }
        }
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            uint32_t bits = 0, word = 0;  // neighbours often share a word: one atomic for them
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const uint32_t g = static_cast<uint32_t>(page[x][y]);
                if (y >= have[x] || g >= a.page_count) continue;
                if (bits != 0 && g / 32 != word) {
                    atomicOr(&used[word], bits);
                    bits = 0;
                }
                word = g / 32;
                bits |= 1u << (g % 32);
            }
            if (bits != 0) atomicOr(&used[word], bits);
        }
    }
    if (a.d.kept != nullptr)
        for (uint32_t p0 = tid; p0 < a.page_count; p0 += kEach * THREADS) {
            uint8_t kept[kEach];
#pragma unroll
            for (int x = 0; x < kEach; ++x) kept[x] = a.d.kept[min(p0 + x * THREADS, a.page_count - 1)];
#pragma unroll
            for (int x = 0; x < kEach; ++x) {
                const uint32_t p = min(p0 + x * THREADS, a.page_count - 1);
                if (kept[x] != 0) atomicOr(&used[p / 32], 1u << (p % 32));
            }
        }
    __syncthreads();
}
// The first `given` pages whose bits are not set, in order: how many there are.
template <int THREADS>
__device__ __forceinline__ uint32_t find_free(const ForkArgs &a, uint32_t given, const uint32_t *used, uint32_t *totals, int32_t *free) {
    const int tid = threadIdx.x, words = static_cast<int>((a.page_count + 31) / 32);
    uint32_t all;
    uint32_t found = 0;
    for (int w0 = 0; w0 < words && found < given; w0 += THREADS) {
        const int w = w0 + tid;
        uint32_t open = w < words ? ~used[w] : 0;
        if (w == words - 1 && a.page_count % 32 != 0) open &= (1u << (a.page_count % 32)) - 1u;
        uint32_t at = found + threads_before<THREADS>(static_cast<uint32_t>(__builtin_popcount(open)), totals, &all);
        found += all;
        for (; open != 0 && at < given; open &= open - 1, ++at) free[at] = 32 * w + __builtin_ctz(open);
    }
    return min(found, given);
}

__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(const ForkArgs a) {
    __shared__ int32_t parent[Q4RDNA_FORK_MAX_SEQUENCES], past[Q4RDNA_FORK_MAX_SEQUENCES];
    __shared__ int32_t first[Q4RDNA_FORK_MAX_SEQUENCES];  // the first that goes on from a sequence
    __shared__ int32_t vacant[Q4RDNA_FORK_MAX_SEQUENCES];  // slots of those that nobody goes on from
    __shared__ int32_t old_past[Q4RDNA_FORK_MAX_SEQUENCES], old_slot[Q4RDNA_FORK_MAX_SEQUENCES];
    __shared__ uint32_t used[kForkPages / 32];
    __shared__ uint32_t totals[kPlanThreads / 64], copies, longest;
    const int tid = threadIdx.x, n = static_cast<int>(a.d.sequences), width = static_cast<int>(a.d.table_width);
    const int words = static_cast<int>((a.page_count + 31) / 32);
    const auto fault = [&] {
        if (a.faults != nullptr) atomicAdd(a.faults, 1u);
    };
    for (int w = tid; w < words; w += kPlanThreads) used[w] = 0;
    for (int i = tid; i < n; i += kPlanThreads) {
        first[i] = n;
        parent[i] = a.d.parents[i];
        old_past[i] = a.d.past[i];
        old_slot[i] = a.d.slots[i];
    }
    if (tid == 0) copies = longest = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kPlanThreads) {
        int p = parent[i], length = 0;
        if (p != -1) {
            bool ok = static_cast<uint32_t>(p) < static_cast<uint32_t>(n);
            if (ok) {
                length = old_past[p];
                ok = length >= 0 && length <= static_cast<int64_t>(width) * kBlock && static_cast<uint32_t>(old_slot[p]) < a.slot_count;
            }
            if (!ok) {
                fault();
                p = -1;
                length = 0;
            }
        }
        parent[i] = p;
        past[i] = length;
        if (p >= 0) atomicMin(&first[p], i);
    }
    __syncthreads();
    uint32_t base = 0, all;
    for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
        const int i = i0 + tid;
        const bool none = i < n && first[i] == n;
        const uint32_t at = base + threads_before<kPlanThreads>(none, totals, &all);
        if (none) vacant[at] = old_slot[i];
        base += all;
    }
    __syncthreads();
    uint32_t later = 0, given = 0;  // as many later children and dropped ones as vacant slots
    for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
        const int i = i0 + tid;
        int p = i < n ? parent[i] : -1, length = i < n ? past[i] : 0;
        const bool moved = i < n && (p < 0 || first[p] != i);
        const uint32_t at = later + threads_before<kPlanThreads>(moved, totals, &all);
        later += all;
        const int from = p >= 0 ? old_slot[p] : 0, slot = moved ? vacant[at] : from;
        if (p >= 0 && static_cast<uint32_t>(slot) >= a.slot_count) {
            fault();
            p = -1;
            length = 0;
        }
        const int blocks = p >= 0 ? max(room_end(a.d, length) - length / kBlock, 0) : 0;
        const uint32_t rank = given + threads_before<kPlanThreads>(static_cast<uint32_t>(blocks), totals, &all);
        given += all;
        if (i < n) {
            parent[i] = p;
            past[i] = length;
            a.moves[i] = ForkMove{p, length, slot, rank};
            if (moved && length > 0) a.copies[atomicAdd(&copies, 1u)] = ForkCopy{from, slot, length};
            if (length >= kBlock) atomicMax(&longest, static_cast<uint32_t>(length / kBlock));
        }
    }
    __syncthreads();
    mark_pages<kPlanThreads>(a, longest, parent, past, first, used);
    const uint32_t found = find_free<kPlanThreads>(a, given, used, totals, a.free);
    if (tid == 0) {
        a.counts[0] = copies;
        a.counts[1] = found;
    }
}

// Renames 2^columns_log2 columns: what sequence i becomes is move(i), the pages
// that are given out, `given` of them, are page(rank).
template <int THREADS, typename Move, typename Page>
__device__ __forceinline__ void move_columns(const ForkArgs &a, int column0, uint32_t given, Move move, Page page) {
    constexpr int kEach = kForkEntries / 256;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // or all entries' rows would stay in registers over the caller's loop
    const int n = static_cast<int>(a.d.sequences), width = static_cast<int>(a.d.table_width);
    const int columns = 1 << a.columns_log2;
    int32_t entry[kEach];
#pragma unroll
    for (int x = 0; x < kEach; ++x) {
        const int e = tid + THREADS * x, i = e >> a.columns_log2, b = column0 + (e & (columns - 1));
        entry[x] = -1;
        if (i >= n || b >= width) continue;
        const ForkMove m = move(i);
        const int full = m.past / kBlock;
        if (m.parent < 0) continue;
        if (b < full) {
            entry[x] = a.d.table[static_cast<size_t>(m.parent) * width + b];
        } else if (b < room_end(a.d, m.past)) {
            const uint32_t rank = m.pages + (b - full);
            if (rank < given) entry[x] = page(rank);
            else if (a.faults != nullptr) atomicAdd(a.faults, 1u);
        }
    }
    wait_stores();  // the loads too: all rows have been read
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kEach; ++x) {
        const int e = tid + THREADS * x, i = e >> a.columns_log2, b = column0 + (e & (columns - 1));
        if (i < n && b < width) a.d.table[static_cast<size_t>(i) * width + b] = entry[x];
    }
}

__device__ __forceinline__ void move_table(const ForkArgs &a) {
    const int tid = threadIdx.x, n = static_cast<int>(a.d.sequences);
    move_columns<256>(a, static_cast<int>(blockIdx.x << a.columns_log2), a.counts[1], [&](int i) { return a.moves[i]; },
                 [&](uint32_t rank) { return a.free[rank]; });
    if (blockIdx.x == 0)
        for (int i = tid; i < n; i += 256) {
            const ForkMove m = a.moves[i];
            a.d.past[i] = m.past;
            a.d.slots[i] = m.slot;
        }
}

// One head's planes and token scales of one block: 16 bytes of a thread, kEach
// times.
template <int D>
__device__ __forceinline__ void copy_open(const ForkArgs &a, const ForkCopy *copies, uint32_t unit) {
    constexpr int kEach = 4 * kBlock * D / (16 * 256);
    const int tid = threadIdx.x % 256;
    const uint32_t head = unit % a.kv_heads, rest = unit / a.kv_heads;
    const uint32_t layer = rest / 2 % a.layers;
    const ForkCopy c = copies[rest / 2 / a.layers];
    // the open block, where it holds tokens, or the one before it
    const int block = c.past / kBlock - static_cast<int>(rest % 2);
    if (block < 0 || block * kBlock >= c.past) return;
    const size_t from = (static_cast<size_t>(c.from) * 2 + (block & 1)) * a.kv_heads + head;
    const size_t to = (static_cast<size_t>(c.to) * 2 + (block & 1)) * a.kv_heads + head;
    constexpr size_t kPlanes = 4 * kBlock * D;
    const int8_t *src = a.open[layer] + from * kPlanes + 16 * tid;
    int8_t *dst = a.open[layer] + to * kPlanes + 16 * tid;
    i32x4 v[kEach];
#pragma unroll
    for (int x = 0; x < kEach; ++x) v[x] = load16(src + 4096 * x);
    if (tid < 2 * kBlock / 4) {
        const i32x4 s = load16(a.open_scales[layer] + from * 2 * kBlock + 4 * tid);
        store16(a.open_scales[layer] + to * 2 * kBlock + 4 * tid, s);
    }
#pragma unroll
    for (int x = 0; x < kEach; ++x) store16(dst + 4096 * x, v[x]);
}

template <int D>
__global__ __launch_bounds__(256) void fork_move_kernel(const ForkArgs a) {
    if (blockIdx.x < a.table_units) {
        move_table(a);
        return;
    }
    const uint32_t copiers = gridDim.x - a.table_units;
    const uint64_t units = static_cast<uint64_t>(a.counts[0]) * a.layers * 2 * a.kv_heads;  // fewer than 2^32
    for (uint64_t u = blockIdx.x - a.table_units; u < units; u += copiers) copy_open<D>(a, a.copies, static_cast<uint32_t>(u));
}

// Both in one launch, for up to 256 sequences: every workgroup plans for itself, which
// is three loads side by side and some steps in LDS.  The first one sees to the
// pages and the table, which no other reads, the others copy; and since all
// read the lengths and slots, the last one to have done so writes them.
template <int D, int THREADS>
__global__ __launch_bounds__(THREADS) void fork_kernel(const ForkArgs a) {
    __shared__ int32_t parent[kForkSmall], past[kForkSmall], slot[kForkSmall], first[kForkSmall], vacant[kForkSmall];
    __shared__ int32_t old_past[kForkSmall], old_slot[kForkSmall], free[kForkSmallGiven];
    __shared__ ForkCopy copy[kForkSmall];
    __shared__ uint32_t used[kForkSmallPages / 32], ranks[kForkSmall], totals[THREADS / 64], longest;
    const int tid = threadIdx.x, lane = tid & 63, n = static_cast<int>(a.d.sequences), width = static_cast<int>(a.d.table_width);
    const bool mine = tid < n, first_one = blockIdx.x == 0;
    int p = -1, length = 0;
    if (mine) {
        p = a.d.parents[tid];
        old_past[tid] = a.d.past[tid];
        old_slot[tid] = a.d.slots[tid];
    }
    if (tid < kForkSmall) first[tid] = n;
    if (first_one)
        for (uint32_t w = tid; w < (a.page_count + 31) / 32; w += THREADS) used[w] = 0;
    if (tid == 0) longest = 0;
    __syncthreads();  // with it, the lengths and slots have arrived
    // Arrivals are counted at gates, 128 bytes apart, and the full gates.
    const uint32_t gate = blockIdx.x % kForkGates;
    uint32_t ticket = 0;
    if (tid == 0) ticket = add_agent(a.arrived + 32 * (1 + gate), 1u);
    bool refused = false;
    if (p != -1) {
        bool ok = static_cast<uint32_t>(p) < static_cast<uint32_t>(n);
        if (ok) {
            length = old_past[p];
            ok = length >= 0 && length <= static_cast<int64_t>(width) * kBlock && static_cast<uint32_t>(old_slot[p]) < a.slot_count;
        }
        if (!ok) {
            refused = true;
            p = -1;
            length = 0;
        }
    }
    if (p >= 0) atomicMin(&first[p], tid);
    __syncthreads();
    uint32_t all;
    const bool none = mine && first[tid] == n, moved = mine && (p < 0 || first[p] != tid);
    const uint32_t at = threads_before<THREADS>((none ? 1u : 0u) + (moved ? 1u << 16 : 0u), totals, &all);
    if (none) vacant[at & 0xffffu] = old_slot[tid];
    __syncthreads();
    const int from = p >= 0 ? old_slot[p] : 0, to = moved ? vacant[at >> 16] : from;
    if (p >= 0 && static_cast<uint32_t>(to) >= a.slot_count) {
        refused = true;
        p = -1;
        length = 0;
    }
    const bool copied = moved && length > 0;
    const int blocks = p >= 0 ? max(room_end(a.d, length) - length / kBlock, 0) : 0;
    // (Fewer than 256 copies, and no more pages than the table has entries.)
    const uint32_t rank = threads_before<THREADS>((copied ? 1u : 0u) + (static_cast<uint32_t>(blocks) << 16), totals, &all);
    if (copied) copy[rank & 0xffffu] = ForkCopy{from, to, length};
    if (tid < kForkSmall) {
        parent[tid] = p;
        past[tid] = length;
        slot[tid] = to;
        ranks[tid] = rank >> 16;
    }
    if (first_one && length >= kBlock) atomicMax(&longest, static_cast<uint32_t>(length / kBlock));
    __syncthreads();
    if (tid < 64) {
        const uint32_t here = (gridDim.x - gate + kForkGates - 1) / kForkGates;
        if (static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(ticket))) == here - 1) {
            uint32_t gates = 0;
            if (lane == 0) {
                store_agent(a.arrived + 32 * (1 + gate), 0u);
                gates = add_agent(a.arrived, 1u) + 1;
                if (gates == min(gridDim.x, kForkGates)) store_agent(a.arrived, 0u);
            }
            if (static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(gates))) == min(gridDim.x, kForkGates))
                for (int i = lane; i < n; i += 64) {
                    a.d.past[i] = past[i];
                    a.d.slots[i] = slot[i];
                }
        }
    }
    if (!first_one) {
        const uint32_t units = (all & 0xffffu) * a.layers * 2 * a.kv_heads;  // fewer than 2^32
        constexpr uint32_t kSide = THREADS / 256;  // units side by side
        for (uint32_t u = (blockIdx.x - 1) * kSide + tid / 256; u < units; u += (gridDim.x - 1) * kSide) copy_open<D>(a, copy, u);
        return;
    }
    if (refused && a.faults != nullptr) atomicAdd(a.faults, 1u);
    mark_pages<THREADS>(a, longest, parent, past, first, used);
    const uint32_t given = find_free<THREADS>(a, all >> 16, used, totals, free);
    __syncthreads();
    for (int column = 0; column < width; column += 1 << a.columns_log2)
        move_columns<THREADS>(a, column, given, [&](int i) { return ForkMove{parent[i], past[i], slot[i], ranks[i]}; }, [&](uint32_t r) { return free[r]; });
}

}  // namespace

hipError_t launch_fork_plan(const ForkArgs &a, hipStream_t stream) {
    fork_plan_kernel<<<1, kPlanThreads, 0, stream>>>(a);
    return hipGetLastError();
}

hipError_t launch_fork_move(const ForkArgs &a, uint32_t copiers, hipStream_t stream) {
    auto go = [&](auto kernel) { kernel<<<a.table_units + copiers, 256, 0, stream>>>(a); };
    a.head_dim == 64 ? go(fork_move_kernel<64>) : go(fork_move_kernel<128>);
    return hipGetLastError();
}

hipError_t launch_fork(const ForkArgs &a, uint32_t threads, uint32_t copiers, hipStream_t stream) {
    auto go = [&](auto kernel) { kernel<<<1 + copiers, threads, 0, stream>>>(a); };
    if (threads == 256) a.head_dim == 64 ? go(fork_kernel<64, 256>) : go(fork_kernel<128, 256>);
    else a.head_dim == 64 ? go(fork_kernel<64, 1024>) : go(fork_kernel<128, 1024>);
    return hipGetLastError();
}

}  // namespace q4rdna
