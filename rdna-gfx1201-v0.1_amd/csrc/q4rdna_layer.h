// Internal interface of the decoder-layer operators: the kernels of
// q4rdna_cache.hip (append, read), q4rdna_attend.hip and q4rdna_norm.hip, with
// their entry points in q4rdna_layer.cpp, and those of q4rdna_draft.hip,
// q4rdna_attend_tree.hip, q4rdna_beam.hip and q4rdna_fork.hip, with theirs in
// q4rdna_branch.cpp.  Not part of the C ABI.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stdint.h>

#include "q4rdna.h"

namespace q4rdna {

constexpr uint32_t kKvBlock = Q4RDNA_KV_BLOCK;

// The 16-bit codes' largest magnitude, 127 * 256: code = 256 * high + low with
// low in [-128, 127] keeps high in [-127, 127].
constexpr int kKvCode16 = 32512;
// Below this largest magnitude a token counts as zero: its 16-bit scale and
// the reciprocal of it stay far from the subnormal numbers.
constexpr float kKvZero = 1e-30f;

struct AppendArgs {
    q4rdna_kv_cache cache;
    q4rdna_kv_batch batch;
    q4rdna_kv_append_desc d;
    uint32_t kv_units;  // (sequence, block) places times kv heads
    uint32_t q_units;   // workgroups that rotate q
    uint32_t q_rows;    // rows (token, query head) that each of them takes
    uint32_t heads_magic;  // div_split's for q_heads
    uint32_t wide;      // rows of k, v, q, q_out can be read four elements at a time
};
hipError_t launch_append(const AppendArgs &a, hipStream_t stream);

struct ReadArgs {
    q4rdna_kv_cache cache;
    q4rdna_kv_batch batch;
    q4rdna_kv_rows k, v;
    uint32_t dtype;
    uint32_t units;
    uint32_t wide;      // k and v rows can be written 16 bytes at a time
};
hipError_t launch_read(const ReadArgs &a, hipStream_t stream);

// Places for the (sequence, block) pairs that a step touches.  Sequence i owns
// the places from cu[i] / 64 + 2 i on: cu[i+1] / 64 - cu[i] / 64 + 2 of them,
// enough for the blocks that its tokens touch, so no prefix sum is needed.
inline uint64_t kv_places(const q4rdna_kv_batch &b) {
    return b.cu_tokens == nullptr ? b.sequences : b.tokens / kKvBlock + 2ull * b.sequences;
}

struct AttendArgs {
    q4rdna_kv_cache cache;
    q4rdna_kv_batch batch;
    q4rdna_kv_attend_desc d;
    uint32_t group;       // query heads per kv head
    uint32_t row_groups;  // row groups of the largest sequence
    uint32_t splits;      // the most workgroups that share a row group
    uint32_t target;      // attend_few_kernel: workgroups to deal the blocks to
    uint32_t workgroups;  // attend_few_kernel: workgroups launched
    uint32_t cu_units;    // attend_many_kernel: workgroups per head when every CU has one
    uint32_t few_rows;    // sequences of up to so many rows belong to attend_few_kernel, the others to
                          // attend_many_kernel
    uint32_t wide;        // q rows can be read 16 bytes at a time
    uint32_t wide_out;    // out rows can be written four elements at a time
    float *partials;      // of each workgroup (attend_few_kernel): [row][D], then all the maxima and sums,
                          // [row][2]; of [job][split] (attend_many_kernel): [D][row], then all the
                          // maxima, sums and units, [3][row]
    uint32_t *arrived;    // [job], zero between launches
};
// The most workgroups that share a row group of attend_few_kernel.
constexpr uint32_t kAttendFewSplits = 64;
// Up to so many blocks are not split, and more than so many are a long row.
constexpr uint32_t kAttendWhole = 16;
constexpr uint32_t kAttendLong = 160;
// Rows (query token, query head of the kv head) that one workgroup takes.
uint32_t attend_few_rows(uint32_t rows);
// waves: 4 or 8 per workgroup.
hipError_t launch_attend_few(const AttendArgs &a, uint32_t rows, uint32_t waves, hipStream_t stream);

// Row groups of 128 (attend_many_kernel) that the step's sequences may have.
constexpr uint32_t kAttendManyRows = 128;
uint64_t attend_many_places(const q4rdna_kv_batch &b, uint32_t group);
hipError_t launch_attend_many(const AttendArgs &a, uint32_t places, hipStream_t stream);

hipError_t launch_add_norm(const q4rdna_add_norm_desc &d, bool wide, uint32_t cus, hipStream_t stream);

constexpr uint32_t kTreeMax = Q4RDNA_TREE_MAX;
hipError_t launch_tree(const q4rdna_kv_batch &batch, const int32_t *parents, int32_t *positions, uint64_t *seen,
                       hipStream_t stream);

struct RotateArgs {
    q4rdna_rotate_desc d;
    uint32_t heads;        // of q and k together
    uint32_t heads_magic;  // div_split's
    uint32_t rows;         // (token, head), fewer than 2^31
    uint32_t unit_rows;    // that a workgroup takes
    uint32_t wide;         // rows can be read and written four elements at a time
};
hipError_t launch_rotate(const RotateArgs &a, hipStream_t stream);

// Rows (query token, query head of a kv head) of a workgroup of
// attend_tree_kernel, a tile, and the most workgroups that share them.
constexpr uint32_t kTreeRows = 32;
constexpr uint32_t kTreeSplits = 64;
struct TreeJob {
    uint32_t first;   // workgroup of a tile's first part
    uint32_t splits;
};
struct TreeArgs {
    q4rdna_kv_cache cache;
    q4rdna_kv_batch batch;
    q4rdna_kv_tree_desc d;
    uint32_t group;       // query heads per kv head
    uint32_t group_magic; // div_split's
    uint32_t tiles;       // of the largest sequence
    uint32_t splits;      // the most workgroups that share a tile
    uint32_t cus;         // to deal the units to
    uint32_t per_cu;      // workgroups that a CU takes
    uint32_t workgroups;  // launched
    float *partials;      // of each workgroup [row][D], then of each [m, l, e][row]
    TreeJob *jobs;        // [sequence][tile][head]
};
hipError_t launch_attend_tree(const TreeArgs &a, hipStream_t stream);

constexpr uint32_t kBeamTrip = 4096;
constexpr uint32_t kBeamPartials = 4;  // sums of a chunk, one of each wave
struct BeamArgs {
    q4rdna_beam_desc d;
    uint32_t trips;     // of a workgroup, kBeamTrip numbers each
    uint32_t chunks;    // of trips * kBeamTrip numbers, per row
    uint64_t *tops;     // [group][count][beam][chunk]: ordered logit << 32 | ~token, 0: none
    uint64_t *stats;    // [group][beam][chunk][kBeamPartials][2]: sum (double), max (float)
    uint32_t *arrived;  // [group], zero between launches
};
hipError_t launch_beam(const BeamArgs &a, hipStream_t stream);

// A sequence's new state, by the plan that fork_plan_kernel makes.
struct ForkMove {
    int32_t parent;  // -1: dropped
    int32_t past;
    int32_t slot;
    uint32_t pages;  // of the pages given out, its first one's rank
};
struct ForkCopy {
    int32_t from, to;  // slots
    int32_t past;
};
// Layers whose open blocks one launch copies.
constexpr uint32_t kForkLayers = 64;
struct ForkArgs {
    q4rdna_kv_fork_desc d;
    uint32_t *faults;
    uint32_t page_count, slot_count, kv_heads, head_dim;
    ForkMove *moves;   // [sequences]
    ForkCopy *copies;  // [sequences]
    uint32_t *counts;  // copies, pages in `free`
    int32_t *free;     // pages in the order in which they are given out
    uint32_t *arrived; // launch_fork's, 32 * (1 + kForkGates) zeros
    uint32_t columns_log2;  // of the table, that a workgroup takes
    uint32_t table_units;
    uint32_t layers;
    int8_t *open[kForkLayers];
    float *open_scales[kForkLayers];
};
// The most pages: their bits lie in LDS.
constexpr uint32_t kForkPages = 1u << 18;
// Entries of the table that a workgroup of 256 threads takes.
constexpr uint32_t kForkEntries = 4096;
// What one launch does: sequences, pages, pages given out at most.
constexpr uint32_t kForkSmall = 256;
constexpr uint32_t kForkSmallPages = 1u << 16;
constexpr uint32_t kForkSmallGiven = 1024;
constexpr uint32_t kForkGates = 16;
// One workgroup for the table and `copiers` for the open blocks, of 256 or 1024
// threads.
hipError_t launch_fork(const ForkArgs &a, uint32_t threads, uint32_t copiers, hipStream_t stream);
hipError_t launch_fork_plan(const ForkArgs &a, hipStream_t stream);
// a.table_units workgroups for the table, the lengths and the slots, and
// `copiers` for the open blocks.
hipError_t launch_fork_move(const ForkArgs &a, uint32_t copiers, hipStream_t stream);

}  // namespace q4rdna
