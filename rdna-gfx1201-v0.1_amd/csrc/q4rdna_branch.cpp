// Entry points of the operators for several continuations of a sequence
// (include/q4rdna.h): argument checks, scratch and the launches.  All compute
// runs in the kernels of q4rdna_draft.hip, q4rdna_attend_tree.hip,
// q4rdna_beam.hip and q4rdna_fork.hip.
#include <algorithm>
#include <cmath>

#include "q4rdna_layer_host.h"

namespace {

using namespace q4rdna;

int current_device(int *device) {
    return hipGetDevice(device) == hipSuccess ? Q4RDNA_OK : set_error(Q4RDNA_ERR_HIP, "no current device");
}

// div_split's for divisors up to 2^16.
uint32_t magic_of(uint32_t d) { return d > 1 ? static_cast<uint32_t>(((1ull << 32) + d - 1) / d) : 0; }

int check_tree_batch(const q4rdna_kv_batch *b) {
    const int rc = check_batch(b);
    if (rc != Q4RDNA_OK || b->sequences == 0 || b->tokens == 0) return rc;
    if (b->max_tokens > kTreeMax)
        return set_error(Q4RDNA_ERR_ARGUMENT, "max_tokens is %u: a tree holds up to %u", b->max_tokens, kTreeMax);
    return Q4RDNA_OK;
}

int tree(const q4rdna_kv_batch *batch, const int32_t *parents, int32_t *positions, uint64_t *seen, void *stream) {
    if (const int rc = check_tree_batch(batch); rc != Q4RDNA_OK) return rc;
    if (batch->sequences == 0 || batch->tokens == 0) return Q4RDNA_OK;
    if (parents == nullptr || positions == nullptr || seen == nullptr)
        return set_error(Q4RDNA_ERR_ARGUMENT, "null parents, positions or seen");
    if (!aligned(parents, 4) || !aligned(positions, 4) || !aligned(seen, 8))
        return set_error(Q4RDNA_ERR_ARGUMENT, "misaligned parents, positions or seen");
    return launched(launch_tree(*batch, parents, positions, seen, static_cast<hipStream_t>(stream)), "kv_tree");
}

int rotate(const q4rdna_rotate_desc *desc, void *stream) {
    if (desc == nullptr) return set_error(Q4RDNA_ERR_ARGUMENT, "null descriptor");
    const q4rdna_rotate_desc &d = *desc;
    int rc;
    if ((rc = check_dtype(d.dtype)) != Q4RDNA_OK) return rc;
    if (d.head_dim != 64 && d.head_dim != 128)
        return set_error(Q4RDNA_ERR_ARGUMENT, "head_dim is %u: 64 and 128 are supported", d.head_dim);
    if (d.reserved != 0) return set_error(Q4RDNA_ERR_ARGUMENT, "reserved is not zero");
    const uint64_t heads = static_cast<uint64_t>(d.q_heads) + d.k_heads, rows = heads * d.tokens;
    if (heads > 32768 || rows > 0x7fffffffu)
        return set_error(Q4RDNA_ERR_ARGUMENT, "%u tokens of %u and %u heads", d.tokens, d.q_heads, d.k_heads);
    if (rows == 0) return Q4RDNA_OK;
    if (d.q_heads != 0 && ((rc = check_rows(d.q, d.dtype, "q")) != Q4RDNA_OK || (rc = check_rows(d.q_out, d.dtype, "q_out")) != Q4RDNA_OK))
        return rc;
    if (d.k_heads != 0 && ((rc = check_rows(d.k, d.dtype, "k")) != Q4RDNA_OK || (rc = check_rows(d.k_out, d.dtype, "k_out")) != Q4RDNA_OK))
        return rc;
    if (d.rotary % 8 != 0 || d.rotary > d.head_dim)
        return set_error(Q4RDNA_ERR_ARGUMENT, "rotary is %u: a multiple of 8 up to head_dim is needed", d.rotary);
    if (d.rotary != 0) {
        if (d.cos == nullptr || d.sin == nullptr || d.positions == 0 || !aligned(d.cos, 16) || !aligned(d.sin, 16))
            return set_error(Q4RDNA_ERR_ARGUMENT, "cos and sin have to be 16-byte aligned tables");
        if (d.position == nullptr || !aligned(d.position, 4)) return set_error(Q4RDNA_ERR_ARGUMENT, "null or misaligned position");
    }
    if (!aligned(d.q_norm, 16) || !aligned(d.k_norm, 16)) return set_error(Q4RDNA_ERR_ARGUMENT, "misaligned norm weight");
    RotateArgs a{};
    a.d = d;
    a.heads = static_cast<uint32_t>(heads);
    a.heads_magic = magic_of(a.heads);
    a.rows = static_cast<uint32_t>(rows);
    // A row for each group of lanes of a workgroup, or two where there are many (61 MB:
    // one 17.1 us, two 16.1, four 16.3, eight 17.5).
    a.unit_rows = rows <= 4096 ? 2048 / d.head_dim : 4096 / d.head_dim;
    a.wide = (d.q_heads == 0 || (wide_rows(d.q, d.dtype, 4) && wide_rows(d.q_out, d.dtype, 4))) &&
             (d.k_heads == 0 || (wide_rows(d.k, d.dtype, 4) && wide_rows(d.k_out, d.dtype, 4)));
    if ((rows + a.unit_rows - 1) / a.unit_rows > most_workgroups(256))
        return set_error(Q4RDNA_ERR_ARGUMENT, "%u tokens are too many for one call", d.tokens);
    return launched(launch_rotate(a, static_cast<hipStream_t>(stream)), "rotate");
}

// Up to so many sequences the blocks are dealt by their lengths, as in
// q4rdna_kv_attend.
constexpr uint32_t kDealtSequences = 256;

int attend_tree(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch, const q4rdna_kv_tree_desc *desc, void *stream) {
    int rc;
    if ((rc = check_cache(cache)) != Q4RDNA_OK || (rc = check_tree_batch(batch)) != Q4RDNA_OK) return rc;
    if (desc == nullptr) return set_error(Q4RDNA_ERR_ARGUMENT, "null descriptor");
    if (batch->sequences == 0 || batch->tokens == 0) return Q4RDNA_OK;
    const q4rdna_kv_tree_desc &d = *desc;
    if ((rc = check_dtype(d.dtype)) != Q4RDNA_OK || (rc = check_heads(d.q_heads, cache->kv_heads)) != Q4RDNA_OK ||
        (rc = check_rows(d.q, d.dtype, "q")) != Q4RDNA_OK || (rc = check_rows(d.k, d.dtype, "k")) != Q4RDNA_OK ||
        (rc = check_rows(d.v, d.dtype, "v")) != Q4RDNA_OK || (rc = check_rows(d.out, d.dtype, "out")) != Q4RDNA_OK)
        return rc;
    if (d.seen == nullptr || !aligned(d.seen, 8)) return set_error(Q4RDNA_ERR_ARGUMENT, "null or misaligned seen");
    if (!std::isfinite(d.scale) || d.scale < 0.0f)
        return set_error(Q4RDNA_ERR_ARGUMENT, "scale is %g: a finite number >= 0 is needed", static_cast<double>(d.scale));
    if (!aligned(d.lse, 4)) return set_error(Q4RDNA_ERR_ARGUMENT, "misaligned lse");
    TreeArgs a{};
    a.cache = *cache;
    a.batch = *batch;
    a.d = d;
    a.group = d.q_heads / cache->kv_heads;
    a.group_magic = magic_of(a.group);
    // The most rows (query token, query head) per kv head that a sequence has.
    const uint32_t most_rows = std::min(batch->max_tokens, batch->tokens) * a.group;
    a.tiles = (most_rows + kTreeRows - 1) / kTreeRows;
    const uint64_t jobs = static_cast<uint64_t>(a.tiles) * cache->kv_heads * batch->sequences;
    const uint64_t most_units = (d.window == 0 ? batch->table_width
                                               : std::min<uint64_t>(batch->table_width, d.window / kKvBlock + 2)) + 3ull;
    const uint32_t cus = cu_count(cache->device);
    a.cus = cus;
    // (Parts are not worth their scratch where tiles abound, nor a second launch
    // where a wave has four units at most.)
    const bool split = most_units > 16 && batch->sequences <= kDealtSequences && jobs <= 16ull * cus && jobs * most_units <= 0x7fffffffu;
    a.splits = static_cast<uint32_t>(split ? std::min<uint64_t>((most_units + 3) / 4, kTreeSplits) : 1);
    // (Blocks by the tables' width.  With one, fp32 needs no scratch: 1% for a few
    // tokens; with two, more tiles than CUs share them.)
    const bool many = jobs * most_units > 31ull * cus;
    a.per_cu = jobs > cus || many ? 2 : 1;
    const uint64_t workgroups = split ? std::min(jobs + (many ? 2 : 1) * cus, jobs * a.splits) : jobs;
    if (workgroups > most_workgroups(256))
        return set_error(Q4RDNA_ERR_ARGUMENT, "%u sequences of %u kv heads are too many for one call", batch->sequences, cache->kv_heads);
    a.workgroups = static_cast<uint32_t>(workgroups);
    const OnDevice device(cache->device);
    if (device.status() != Q4RDNA_OK) return device.status();
    const hipStream_t s = static_cast<hipStream_t>(stream);
    Scratch scratch;  // held over the launches
    if (a.splits > 1) {
        const size_t floats = workgroups * kTreeRows * (cache->head_dim + 3);
        if ((rc = get_scratch(cache->device, s, floats + 2 * jobs, 0, &scratch)) != Q4RDNA_OK) return rc;
        a.partials = scratch.partials;
        a.jobs = reinterpret_cast<TreeJob *>(scratch.partials + floats);
    }
    return launched(launch_attend_tree(a, s), "kv_attend_tree");
}

int beam_select(const q4rdna_beam_desc *desc, void *stream) {
    if (desc == nullptr) return set_error(Q4RDNA_ERR_ARGUMENT, "null descriptor");
    const q4rdna_beam_desc &d = *desc;
    int rc;
    if ((rc = check_dtype(d.dtype)) != Q4RDNA_OK) return rc;
    if (d.reserved != 0) return set_error(Q4RDNA_ERR_ARGUMENT, "reserved is not zero");
    if (d.beams == 0 || d.beams > Q4RDNA_BEAM_MAX_BEAMS || d.vocab == 0 || d.vocab > (1u << 24) ||
        static_cast<uint64_t>(d.groups) * d.beams > 0x7fffffffu)
        return set_error(Q4RDNA_ERR_ARGUMENT, "%u groups of %u beams over %u tokens", d.groups, d.beams, d.vocab);
    if (d.count == 0 || d.count > Q4RDNA_BEAM_MAX_COUNT || d.count > static_cast<uint64_t>(d.beams) * d.vocab)
        return set_error(Q4RDNA_ERR_ARGUMENT, "count is %u: 1 to %d, and no more than there are continuations", d.count,
                         Q4RDNA_BEAM_MAX_COUNT);
    if (d.groups == 0) return Q4RDNA_OK;
    if (d.logits == nullptr || d.out_scores == nullptr || d.out_rows == nullptr || d.out_tokens == nullptr)
        return set_error(Q4RDNA_ERR_ARGUMENT, "null logits or output");
    if (!aligned(d.logits, size_of(d.dtype)) || !aligned(d.scores, 4) || !aligned(d.out_scores, 4) || !aligned(d.out_rows, 4) ||
        !aligned(d.out_tokens, 4))
        return set_error(Q4RDNA_ERR_ARGUMENT, "misaligned buffer");
    int device = 0;
    if ((rc = current_device(&device)) != Q4RDNA_OK) return rc;
    BeamArgs a{};
    a.d = d;
    // A trip costs a workgroup 0.8 us, its own start and end 4, and every chunk's
    // items lengthen the join: up to three workgroups a CU, and up to 128 chunks of
    // a group, a chunk is one trip (one, two and three trips: 4 rows of 151936 in
    // fp32, 152 trips, 11.7, 11.5, 12.8 us; one row 7.8, 8.8, 9.5; 160 rows of
    // 50257 in bf16, 2080 trips, 36.7, 23.7, 18.3, and 19.3 with four).
    const uint64_t rows = static_cast<uint64_t>(d.groups) * d.beams;
    const uint32_t row_trips = (d.vocab + kBeamTrip - 1) / kBeamTrip;
    const uint64_t most = 3ull * cu_count(device);
    a.trips = static_cast<uint32_t>(std::max<uint64_t>((rows * row_trips + most - 1) / most,
                                                       (static_cast<uint64_t>(d.beams) * row_trips + 127) / 128));
    a.trips = std::min(a.trips, row_trips);
    a.chunks = (row_trips + a.trips - 1) / a.trips;
    const uint64_t lists = rows * a.chunks;
    if (lists > most_workgroups(256) || static_cast<uint64_t>(d.beams) * a.chunks * d.count > 0x7fffffffu)
        return set_error(Q4RDNA_ERR_ARGUMENT, "%u groups of %u beams are too many for one call", d.groups, d.beams);
    Scratch scratch;
    if ((rc = get_scratch(device, static_cast<hipStream_t>(stream), 2 * lists * (d.count + 2 * kBeamPartials), d.groups, &scratch)) != Q4RDNA_OK) return rc;
    a.tops = reinterpret_cast<uint64_t *>(scratch.partials);
    a.stats = a.tops + lists * d.count;
    a.arrived = scratch.arrived;
    return launched(launch_beam(a, static_cast<hipStream_t>(stream)), "beam_select");
}

int fork(const q4rdna_kv_cache *caches, uint32_t count, const q4rdna_kv_fork_desc *desc, void *stream) {
    int rc;
    if (caches == nullptr || count == 0) return set_error(Q4RDNA_ERR_ARGUMENT, "no caches");
    if (desc == nullptr) return set_error(Q4RDNA_ERR_ARGUMENT, "null descriptor");
    const q4rdna_kv_cache &c = caches[0];
    for (uint32_t i = 0; i < count; ++i) {
        if ((rc = check_cache(caches + i)) != Q4RDNA_OK) return rc;
        const q4rdna_kv_cache &o = caches[i];
        if (o.page_count != c.page_count || o.slot_count != c.slot_count || o.kv_heads != c.kv_heads || o.head_dim != c.head_dim ||
            o.device != c.device)
            return set_error(Q4RDNA_ERR_ARGUMENT, "cache %u is of another geometry or device than the first", i);
        for (uint32_t j = 0; j < i; ++j)
            if (caches[j].open == o.open || caches[j].open_scales == o.open_scales)
                return set_error(Q4RDNA_ERR_ARGUMENT, "caches %u and %u share their open blocks", j, i);
    }
    const q4rdna_kv_fork_desc &d = *desc;
    if (d.reserved != 0) return set_error(Q4RDNA_ERR_ARGUMENT, "reserved is not zero");
    if (d.sequences > Q4RDNA_FORK_MAX_SEQUENCES || d.table_width == 0 || d.table_width > (1u << 24))
        return set_error(Q4RDNA_ERR_ARGUMENT, "%u sequences, %u table columns: up to %d and 2^24 are supported", d.sequences,
                         d.table_width, Q4RDNA_FORK_MAX_SEQUENCES);
    if (c.page_count > kForkPages) return set_error(Q4RDNA_ERR_ARGUMENT, "%u pages: up to %u are supported", c.page_count, kForkPages);
    if (d.sequences == 0) return Q4RDNA_OK;
    if (d.parents == nullptr || d.past == nullptr || d.table == nullptr || d.slots == nullptr)
        return set_error(Q4RDNA_ERR_ARGUMENT, "null parents, past, table or slots");
    if (!aligned(d.parents, 4) || !aligned(d.past, 4) || !aligned(d.table, 4) || !aligned(d.slots, 4))
        return set_error(Q4RDNA_ERR_ARGUMENT, "misaligned parents, past, table or slots");
    const OnDevice device(c.device);
    if (device.status() != Q4RDNA_OK) return device.status();
    ForkArgs a{};
    a.d = d;
    a.faults = c.faults;
    a.page_count = c.page_count;
    a.slot_count = c.slot_count;
    a.kv_heads = c.kv_heads;
    a.head_dim = c.head_dim;
    const uint64_t touched = std::min<uint64_t>(d.table_width, static_cast<uint64_t>(d.room) / kKvBlock + 2);
    const uint64_t given = std::min<uint64_t>(c.page_count, touched * d.sequences);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    Scratch scratch;  // held over the launches
    const uint32_t cus = cu_count(c.device);
    const auto take_layers = [&](uint32_t first) {
        a.layers = std::min(count - first, kForkLayers);
        for (uint32_t l = 0; l < a.layers; ++l) {
            a.open[l] = caches[first + l].open;
            a.open_scales[l] = caches[first + l].open_scales;
        }
        // All but one sequence may be copied.
        return static_cast<uint64_t>(d.sequences - 1) * a.layers * 2 * c.kv_heads;
    };
    uint32_t width_log2 = 0;
    while (1u << width_log2 < d.table_width) ++width_log2;
    // One launch where one workgroup can see to the table: in a step, or, with 1024
    // threads, in a few.  A larger table takes many, after a plan.
    const uint64_t entries = static_cast<uint64_t>(d.sequences) << width_log2;
    if (count <= kForkLayers && d.sequences <= kForkSmall && c.page_count <= kForkSmallPages && given <= kForkSmallGiven &&
        entries <= 8 * kForkEntries) {
        if ((rc = get_scratch(c.device, s, 0, 32 * (1 + kForkGates), &scratch)) != Q4RDNA_OK) return rc;
        a.arrived = scratch.arrived;
        const uint32_t threads = entries <= kForkEntries ? 256 : 1024, side = threads / 256;
        while (a.columns_log2 < width_log2 && (d.sequences << (a.columns_log2 + 1)) <= side * kForkEntries) ++a.columns_log2;
        // 1024 threads a CU carry a copy.  (2048 where they wait for each other: 48.5 us,
        // not 49.5, for 200 sequences.)
        const uint64_t most = take_layers(0);
        return launched(launch_fork(a, threads, static_cast<uint32_t>(std::min<uint64_t>((most + side - 1) / side, (side == 1 ? 4 : 2) * cus)), s), "kv_fork");
    }
    if ((rc = get_scratch(c.device, s, 7ull * d.sequences + 2 + given, 0, &scratch)) != Q4RDNA_OK) return rc;
    a.moves = reinterpret_cast<ForkMove *>(scratch.partials);
    a.copies = reinterpret_cast<ForkCopy *>(a.moves + d.sequences);
    a.counts = reinterpret_cast<uint32_t *>(a.copies + d.sequences);
    a.free = reinterpret_cast<int32_t *>(a.counts + 2);
    while (a.columns_log2 < 6 && (d.sequences << (a.columns_log2 + 1)) <= kForkEntries) ++a.columns_log2;
    const uint32_t units = ((d.table_width - 1) >> a.columns_log2) + 1;
    if ((rc = launched(launch_fork_plan(a, s), "kv_fork")) != Q4RDNA_OK) return rc;
    for (uint32_t i = 0; i < count; i += kForkLayers) {
        const uint64_t most = take_layers(i);
        a.table_units = i == 0 ? units : 0;
        // Eight workgroups a CU carry a copy.
        const uint32_t copiers = static_cast<uint32_t>(std::min<uint64_t>(most, 8ull * cus));
        if (a.table_units + copiers == 0) continue;
        if ((rc = launched(launch_fork_move(a, copiers, s), "kv_fork")) != Q4RDNA_OK) return rc;
    }
    return Q4RDNA_OK;
}

}  // namespace

extern "C" {

int q4rdna_kv_tree(const q4rdna_kv_batch *batch, const int32_t *parents, int32_t *positions, uint64_t *seen, void *stream) {
    return guarded([&] { return tree(batch, parents, positions, seen, stream); });
}

int q4rdna_rotate(const q4rdna_rotate_desc *desc, void *stream) {
    return guarded([&] { return rotate(desc, stream); });
}

int q4rdna_kv_attend_tree(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch, const q4rdna_kv_tree_desc *desc,
                          void *stream) {
    return guarded([&] { return attend_tree(cache, batch, desc, stream); });
}

int q4rdna_beam_select(const q4rdna_beam_desc *desc, void *stream) {
    return guarded([&] { return beam_select(desc, stream); });
}

int q4rdna_kv_fork(const q4rdna_kv_cache *caches, uint32_t count, const q4rdna_kv_fork_desc *desc, void *stream) {
    return guarded([&] { return fork(caches, count, desc, stream); });
}

}  // extern "C"
