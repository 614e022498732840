// Entry points of the decoder-layer operators (include/q4rdna.h): argument
// checks, attention's scratch and the launches.  All compute runs in the
// kernels of q4rdna_cache.hip, q4rdna_attend.hip and q4rdna_norm.hip.
#include "q4rdna_layer_host.h"

#include <algorithm>
#include <cmath>
#include <map>
#include <utility>
#include <vector>

namespace q4rdna {
namespace {

// One stream's buffers.  Those that were outgrown are kept.
struct StreamScratch {
    std::mutex mu;
    float *partials = nullptr;
    size_t floats = 0;
    uint32_t *arrived = nullptr;
    size_t jobs = 0;
    std::vector<void *> retired;
};
std::mutex g_scratch_mu;  // of the map: its entries stay where they are
std::map<std::pair<int, hipStream_t>, StreamScratch> g_scratch;

StreamScratch &stream_scratch(int device, hipStream_t stream) {
    std::lock_guard<std::mutex> lock(g_scratch_mu);
    return g_scratch[{device, stream}];
}

bool stream_captured(hipStream_t stream) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream, &status) != hipSuccess) {
        (void)hipGetLastError();
        return false;
    }
    return status == hipStreamCaptureStatusActive;
}

// Device memory while other streams may be under capture: relaxed mode, and
// zeros (where asked for) in the order of the stream.
hipError_t relaxed_malloc(void **p, size_t bytes, bool zero, hipStream_t stream) {
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    hipError_t e = hipThreadExchangeStreamCaptureMode(&mode);
    if (e != hipSuccess) return e;
    e = hipMalloc(p, bytes);
    if (e == hipSuccess && zero && (e = hipMemsetAsync(*p, 0, bytes, stream)) != hipSuccess) (void)hipFree(*p);
    (void)hipThreadExchangeStreamCaptureMode(&mode);
    return e;
}

}  // namespace

int get_scratch(int device, hipStream_t stream, size_t floats, size_t jobs, Scratch *out) {
    StreamScratch &s = stream_scratch(device, stream);
    std::unique_lock<std::mutex> lock(s.mu);
    if (s.floats < floats || s.jobs < jobs) {
        if (stream_captured(stream))
            return set_error(Q4RDNA_ERR_MEMORY, "attention scratch: it cannot grow while its stream is being captured");
        s.retired.reserve(s.retired.size() + 2);
        if (s.floats < floats) {
            const size_t count = std::max(floats, 2 * s.floats);
            void *p = nullptr;
            const hipError_t e = relaxed_malloc(&p, count * sizeof(float), false, stream);
            if (e != hipSuccess) return set_error(Q4RDNA_ERR_MEMORY, "attention scratch: %s", hipGetErrorString(e));
            if (s.partials != nullptr) s.retired.push_back(s.partials);
            s.partials = static_cast<float *>(p);
            s.floats = count;
        }
        if (s.jobs < jobs) {
            const size_t count = std::max(jobs, 2 * s.jobs);
            void *p = nullptr;
            const hipError_t e = relaxed_malloc(&p, count * sizeof(uint32_t), true, stream);
            if (e != hipSuccess) return set_error(Q4RDNA_ERR_MEMORY, "attention scratch: %s", hipGetErrorString(e));
            if (s.arrived != nullptr) s.retired.push_back(s.arrived);
            s.arrived = static_cast<uint32_t *>(p);
            s.jobs = count;
        }
    }
    out->partials = s.partials;
    out->arrived = s.arrived;
    out->held = std::move(lock);
    return Q4RDNA_OK;
}

}  // namespace q4rdna

namespace {

using namespace q4rdna;

int append(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch, const q4rdna_kv_append_desc *desc, void *stream) {
    int rc;
    if ((rc = check_cache(cache)) != Q4RDNA_OK || (rc = check_batch(batch)) != Q4RDNA_OK) return rc;
    if (desc == nullptr) return set_error(Q4RDNA_ERR_ARGUMENT, "null descriptor");
    if (batch->sequences == 0 || batch->tokens == 0) return Q4RDNA_OK;
    if ((rc = check_dtype(desc->dtype)) != Q4RDNA_OK || (rc = check_rows(desc->k, desc->dtype, "k")) != Q4RDNA_OK ||
        (rc = check_rows(desc->v, desc->dtype, "v")) != Q4RDNA_OK)
        return rc;
    if (desc->q_heads != 0 && ((rc = check_heads(desc->q_heads, cache->kv_heads)) != Q4RDNA_OK ||
                               (rc = check_rows(desc->q, desc->dtype, "q")) != Q4RDNA_OK ||
                               (rc = check_rows(desc->q_out, desc->dtype, "q_out")) != Q4RDNA_OK))
        return rc;
    if (desc->rotary % 8 != 0 || desc->rotary > cache->head_dim)
        return set_error(Q4RDNA_ERR_ARGUMENT, "rotary is %u: a multiple of 8 up to head_dim is needed", desc->rotary);
    if (desc->rotary != 0 && (desc->cos == nullptr || desc->sin == nullptr || !aligned(desc->cos, 16) || !aligned(desc->sin, 16)))
        return set_error(Q4RDNA_ERR_ARGUMENT, "cos and sin have to be 16-byte aligned tables");
    if (!aligned(desc->q_norm, 16) || !aligned(desc->k_norm, 16))
        return set_error(Q4RDNA_ERR_ARGUMENT, "misaligned norm weight");
    const uint64_t kv_units = q4rdna::kv_places(*batch) * cache->kv_heads;
    // Few rows of q: one per lane group, so that many workgroups share the
    // wait for them; many: eight, which divides the workgroup's fixed part (32
    // bf16 heads of 128, one against eight: 32 tokens 6.7 and 7.1 us, 128
    // tokens 10.4 and 10.4, 512 tokens 11.6 and 10.8, 2048 tokens 23.1 and 15.4).
    const uint64_t all_rows = static_cast<uint64_t>(batch->tokens) * desc->q_heads;
    const uint32_t q_rows = all_rows <= 4096 ? 2048 / cache->head_dim : 16384 / cache->head_dim;
    const uint64_t q_units = (all_rows + q_rows - 1) / q_rows;
    if (kv_units + q_units > most_workgroups(256)) return set_error(Q4RDNA_ERR_ARGUMENT, "%u tokens are too many for one call", batch->tokens);
    const OnDevice device(cache->device);
    if (device.status() != Q4RDNA_OK) return device.status();
    q4rdna::AppendArgs a{};
    a.cache = *cache;
    a.batch = *batch;
    a.d = *desc;
    a.kv_units = static_cast<uint32_t>(kv_units);
    a.q_units = static_cast<uint32_t>(q_units);
    a.q_rows = q_rows;
    a.heads_magic = desc->q_heads > 1 ? static_cast<uint32_t>(((1ull << 32) + desc->q_heads - 1) / desc->q_heads) : 0;
    a.wide = wide_rows(desc->k, desc->dtype, 4) && wide_rows(desc->v, desc->dtype, 4) &&
             (desc->q_heads == 0 || (wide_rows(desc->q, desc->dtype, 4) && wide_rows(desc->q_out, desc->dtype, 4)));
    return launched(q4rdna::launch_append(a, static_cast<hipStream_t>(stream)), "kv_append");
}

// Sequences of up to so many rows (query token, query head) per kv head go to
// attend_few_kernel, which reads the cache once per eight rows, the others to
// attend_many_kernel, which reads it once per 128 and starts and joins slower.
// Up to 32 rows the former is the faster one or within a tenth; beyond, while
// its row groups all run at once and the blocks that they see are few.  The
// lengths are on the device; the table's width and the window bound them.
// bf16, 8 kv heads, us by the former and the latter:
//   64 rows, one sequence behind 2000 tokens 17 and 26, 8000 28 and 42,
//   30000 59 and 69; 8 sequences behind 500 19 and 27, 8000 108 and 76;
//   16 sequences behind 500 36 and 28.
//   128 rows, one sequence behind 2000 22 and 27, 8000 39 and 43, 30000 103 and
//   72; 4 sequences behind 500 19 and 22, 8000 106 and 50.
uint32_t few_rows(const q4rdna_kv_batch &b, uint32_t group, uint32_t kv_heads, uint64_t most_blocks, uint32_t cus) {
    const auto small = [&](uint32_t rows, uint64_t blocks_per_cu) {
        const uint64_t all = std::min(static_cast<uint64_t>(b.sequences) * rows, static_cast<uint64_t>(b.tokens) * group);
        const uint64_t row_groups = (all + 7) / 8 * kv_heads;
        return row_groups <= 2 * cus && row_groups * most_blocks <= blocks_per_cu * cus;
    };
    return small(128, 64) ? 128 : small(64, 128) ? 64 : 32;
}

// Up to so many sequences the blocks are dealt by their lengths, by a scan of
// all of them in every workgroup; more of them fill the card by themselves (a
// token each of 8 heads, dealt and not, us: 200 of 64 to 4096 tokens 98 and 96,
// 200 of which one has 16000 57 and 100; 400 198 and 178, 133 and 157; 800 420
// and 309, 326 and 224).
constexpr uint32_t kDealtSequences = 256;

int attend(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch, const q4rdna_kv_attend_desc *desc, void *stream) {
    int rc;
    if ((rc = check_cache(cache)) != Q4RDNA_OK || (rc = check_batch(batch)) != Q4RDNA_OK) return rc;
    if (desc == nullptr) return set_error(Q4RDNA_ERR_ARGUMENT, "null descriptor");
    if (batch->sequences == 0 || batch->tokens == 0) return Q4RDNA_OK;
    if ((rc = check_dtype(desc->dtype)) != Q4RDNA_OK || (rc = check_heads(desc->q_heads, cache->kv_heads)) != Q4RDNA_OK ||
        (rc = check_rows(desc->q, desc->dtype, "q")) != Q4RDNA_OK || (rc = check_rows(desc->out, desc->dtype, "out")) != Q4RDNA_OK)
        return rc;
    if (!std::isfinite(desc->scale) || desc->scale < 0.0f)
        return set_error(Q4RDNA_ERR_ARGUMENT, "scale is %g: a finite number >= 0 is needed", static_cast<double>(desc->scale));
    if (!aligned(desc->lse, 4)) return set_error(Q4RDNA_ERR_ARGUMENT, "misaligned lse");
    q4rdna::AttendArgs a{};
    a.cache = *cache;
    a.batch = *batch;
    a.d = *desc;
    a.group = desc->q_heads / cache->kv_heads;
    a.wide = wide_rows(desc->q, desc->dtype, 16 / size_of(desc->dtype));
    a.wide_out = wide_rows(desc->out, desc->dtype, 4);
    // The most rows (query token, query head) per kv head that a sequence has.
    const uint64_t most_tokens = std::min(batch->max_tokens, batch->tokens), most_rows = most_tokens * a.group;
    const uint64_t places = q4rdna::attend_many_places(*batch, a.group), many_jobs = places * cache->kv_heads;
    const uint32_t cus = cu_count(cache->device);
    const uint64_t most_blocks = desc->window == 0 ? batch->table_width
                                                   : std::min<uint64_t>(batch->table_width, (desc->window + most_tokens) / q4rdna::kKvBlock + 2);
    const uint32_t few = few_rows(*batch, a.group, cache->kv_heads, most_blocks, cus);
    const bool many = most_rows > few;
    if (most_rows > 0x3fffffffu || (many && many_jobs > most_workgroups(256)))
        return set_error(Q4RDNA_ERR_ARGUMENT, "%u tokens of %u query heads are too many for one call", batch->tokens, desc->q_heads);
    // Both launches are planned and their scratch is there before the first of
    // them, so a call that is refused has launched nothing.
    size_t floats = 0, jobs = 0;  // room for the parts' rows and the statistics beside them; row groups
    q4rdna::AttendArgs f = a, m = a;
    // Sequences of few rows; a single one goes by the bound alone.
    uint32_t rows = 0, waves = 0;
    if (!many || batch->sequences > 1) {
        f.few_rows = many ? few : 0x7fffffffu;
        const uint32_t most = static_cast<uint32_t>(many ? few : most_rows);
        rows = q4rdna::attend_few_rows(most);
        f.row_groups = (most + rows - 1) / rows;
        // The device deals the blocks to about `target` workgroups; each row
        // group ends in one part that may be short.
        const uint64_t few_jobs = static_cast<uint64_t>(f.row_groups) * cache->kv_heads * batch->sequences;
        // Few row groups are cut into many parts, which cost time to join: take
        // one workgroup of eight waves per CU there, two of four waves elsewhere
        // (eight and four waves: one token behind 60000 30.7 and 33.1 us, 32
        // ragged sequences of 100 to 8000 tokens 30.9 and 27.2 us).
        waves = few_jobs < cus / 8 ? 8 : 4;
        f.target = 8 / waves * cus;
        const uint64_t most_splits = (most_blocks + 7) / 8;
        // (Nor are parts worth their scratch where row groups abound.)
        const bool split = most_blocks > q4rdna::kAttendWhole && batch->sequences <= kDealtSequences && few_jobs <= 64ull * cus;
        f.splits = static_cast<uint32_t>(split ? std::min<uint64_t>(most_splits, q4rdna::kAttendFewSplits) : 1);
        const uint64_t workgroups = split ? std::min(few_jobs + f.target, few_jobs * f.splits) : few_jobs;
        if (workgroups > most_workgroups(64 * waves))
            return set_error(Q4RDNA_ERR_ARGUMENT, "%u sequences of %u kv heads are too many for one call", batch->sequences, cache->kv_heads);
        f.workgroups = static_cast<uint32_t>(workgroups);
        if (f.splits > 1) {
            floats = workgroups * rows * (cache->head_dim + 2);
            jobs = few_jobs;
        }
    }
    if (many) {
        m.few_rows = batch->sequences > 1 ? few : 0;
        // Two workgroups fit a CU: split until they are there.
        const uint64_t splits = std::min<uint64_t>(2ull * cus / many_jobs, (most_blocks + 1) / 2);
        m.splits = static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(splits, 64)));
        m.cu_units = std::max(1u, cus / cache->kv_heads);
        if (m.splits > 1) {
            floats = std::max<size_t>(floats, many_jobs * m.splits * q4rdna::kAttendManyRows * (cache->head_dim + 3));
            jobs = std::max<size_t>(jobs, many_jobs);
        }
    }
    const OnDevice device(cache->device);
    if (device.status() != Q4RDNA_OK) return device.status();
    const hipStream_t s = static_cast<hipStream_t>(stream);
    Scratch scratch;  // held over the launches
    if (jobs != 0) {
        if ((rc = get_scratch(cache->device, s, floats, jobs, &scratch)) != Q4RDNA_OK) return rc;
        f.partials = m.partials = scratch.partials;
        f.arrived = m.arrived = scratch.arrived;
    }
    if (rows != 0 && (rc = launched(q4rdna::launch_attend_few(f, rows, waves, s), "kv_attend")) != Q4RDNA_OK) return rc;
    return many ? launched(q4rdna::launch_attend_many(m, static_cast<uint32_t>(places), s), "kv_attend") : Q4RDNA_OK;
}

int read(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch, uint32_t dtype, const q4rdna_kv_rows *k,
         const q4rdna_kv_rows *v, void *stream) {
    int rc;
    if ((rc = check_cache(cache)) != Q4RDNA_OK || (rc = check_batch(batch)) != Q4RDNA_OK) return rc;
    if (k == nullptr || v == nullptr) return set_error(Q4RDNA_ERR_ARGUMENT, "null rows");
    if (batch->sequences == 0 || batch->tokens == 0) return Q4RDNA_OK;
    if ((rc = check_dtype(dtype)) != Q4RDNA_OK || (rc = check_rows(*k, dtype, "k")) != Q4RDNA_OK ||
        (rc = check_rows(*v, dtype, "v")) != Q4RDNA_OK)
        return rc;
    const uint64_t units = q4rdna::kv_places(*batch) * cache->kv_heads;
    if (units > most_workgroups(256)) return set_error(Q4RDNA_ERR_ARGUMENT, "%u tokens are too many for one call", batch->tokens);
    const OnDevice device(cache->device);
    if (device.status() != Q4RDNA_OK) return device.status();
    q4rdna::ReadArgs a{};
    a.cache = *cache;
    a.batch = *batch;
    a.k = *k;
    a.v = *v;
    a.dtype = dtype;
    a.units = static_cast<uint32_t>(units);
    a.wide = wide_rows(*k, dtype, 16 / size_of(dtype)) && wide_rows(*v, dtype, 16 / size_of(dtype));
    return launched(q4rdna::launch_read(a, static_cast<hipStream_t>(stream)), "kv_read");
}

int add_norm(const q4rdna_add_norm_desc *desc, void *stream) {
    if (desc == nullptr) return set_error(Q4RDNA_ERR_ARGUMENT, "null descriptor");
    const q4rdna_add_norm_desc &d = *desc;
    int rc;
    if ((rc = check_dtype(d.dtype)) != Q4RDNA_OK) return rc;
    if (d.width == 0 || d.width > Q4RDNA_NORM_MAX_WIDTH || d.rows > 0x7fffffffu)
        return set_error(Q4RDNA_ERR_ARGUMENT, "%u rows of %u: 1 to %d numbers a row are supported", d.rows, d.width,
                         Q4RDNA_NORM_MAX_WIDTH);
    if (d.rows == 0 || (d.h == nullptr && d.n == nullptr)) return Q4RDNA_OK;
    if (d.residual == nullptr) return set_error(Q4RDNA_ERR_ARGUMENT, "null residual");
    if (d.n != nullptr && d.weight == nullptr) return set_error(Q4RDNA_ERR_ARGUMENT, "n needs a weight");
    if (d.y == nullptr && (d.gate != nullptr || d.post_weight != nullptr))
        return set_error(Q4RDNA_ERR_ARGUMENT, "a gate or a norm of y without y");
    if (d.reserved != 0) return set_error(Q4RDNA_ERR_ARGUMENT, "reserved is not zero");
    const uint32_t size = size_of(d.dtype);
    const void *const buffers[] = {d.residual, d.y, d.gate, d.h, d.n};
    const int64_t strides[] = {d.residual_stride, d.y_stride, d.gate_stride, d.h_stride, d.n_stride};
    bool wide = d.width % (16 / size) == 0 && aligned(d.weight, 16) && aligned(d.post_weight, 16);
    for (int i = 0; i < 5; ++i) {
        if (!aligned(buffers[i], size)) return set_error(Q4RDNA_ERR_ARGUMENT, "misaligned buffer");
        if (buffers[i] != nullptr) wide = wide && aligned(buffers[i], 16) && strides[i] % (16 / size) == 0;
    }
    if (!aligned(d.weight, 4) || !aligned(d.post_weight, 4)) return set_error(Q4RDNA_ERR_ARGUMENT, "misaligned weight");
    if (d.h == d.n) return set_error(Q4RDNA_ERR_ARGUMENT, "h and n are one buffer");
    for (int o = 3; o < 5; ++o)
        for (int i = 0; i < 3; ++i)
            if (d.rows > 1 && buffers[o] != nullptr && buffers[o] == buffers[i] && (strides[o] != strides[i] || i == 2))
                return set_error(Q4RDNA_ERR_ARGUMENT, "an output over an input with another stride, or over the gate");
    int device = 0;
    if (hipGetDevice(&device) != hipSuccess) return set_error(Q4RDNA_ERR_HIP, "no current device");
    return launched(q4rdna::launch_add_norm(d, wide, cu_count(device), static_cast<hipStream_t>(stream)), "add_norm");
}

}  // namespace

extern "C" {

int q4rdna_kv_append(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch, const q4rdna_kv_append_desc *desc,
                     void *stream) {
    return guarded([&] { return append(cache, batch, desc, stream); });
}

int q4rdna_kv_attend(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch, const q4rdna_kv_attend_desc *desc,
                     void *stream) {
    return guarded([&] { return attend(cache, batch, desc, stream); });
}

int q4rdna_kv_read(const q4rdna_kv_cache *cache, const q4rdna_kv_batch *batch, uint32_t dtype, const q4rdna_kv_rows *k,
                   const q4rdna_kv_rows *v, void *stream) {
    return guarded([&] { return read(cache, batch, dtype, k, v, stream); });
}

int q4rdna_add_norm(const q4rdna_add_norm_desc *desc, void *stream) {
    return guarded([&] { return add_norm(desc, stream); });
}

}  // extern "C"
