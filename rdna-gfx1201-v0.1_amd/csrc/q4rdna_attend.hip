// Attention over the 8-bit paged cache (q4rdna_kv_attend).
//
// attend_few_kernel: few rows (query token, query head) per kv head, the
// decode form.  It streams the cache once and multiplies by the int8 codes as
// they lie in memory, with no conversion:
//
//  * A row of q becomes 32-bit fixed point relative to its largest number, as
//    four balanced base-256 digits, so q . k is four int8 dot products, exact
//    in int32.  The digits of four rows fill the 16 columns of a 16x16x64 int8
//    matrix instruction (column 4 r + digit), which is what a group of four
//    query heads needs; a tile of K is its other operand straight from memory.
//  * Its results S^T lie as (token, column): the four lanes of a quad hold a
//    row's digits, two DPP adds join them, and each lane then holds 16 of the
//    64 scores of its row -- in the k order that the second product's operand
//    has, so the weights p never leave their lanes.  They become 30-bit fixed
//    point relative to the block's largest and the lane keeps its digit's byte.
//  * O^T += V^T p by the same instruction, and each lane scales its digit's
//    int32 sums into fp32 accumulators (the digits are joined once at the end).
//
// Each wave keeps its own running maximum and sum (base 2) over the blocks it
// takes; a workgroup's waves, then the workgroups that share a row group,
// are joined by those.  The last workgroup to arrive joins them, in a fixed
// order, so results do not depend on the order of arrival.
//
// The digits make the products four times as many, and the matrix unit is
// still idle nine tenths of the time: a single token is bound by the cache's
// bytes.  130000 tokens behind one (8 kv heads of four query heads of 128
// numbers, 266 MB) take 54.5 us, 4.9 TB/s: 2 us to deal the blocks, 5 until the
// first tiles arrive, 37 at 7.2 TB/s, a plain read's rate, then waiting for the
// slowest workgroups and the join.  Eight query heads a kv head take 65 us.
// A row group is cut into 64 parts at most (one trip joins them), so a single
// sequence of one to three kv heads leaves CUs idle.  With a short cache the chain
// of dependent loads (lengths, page, codes, the open block's V behind its softmax)
// is what is left: 6.4 us behind 17 tokens.
//
// Eight or four waves a workgroup and two waves per SIMD, 185 registers each
// (256 for eight rows): both operands of a block and its accumulators stay in
// registers, nothing goes through LDS but the joins.  Three waves per SIMD
// would spill, and were slower.
#include "q4rdna_layer_device.h"

namespace q4rdna {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
constexpr int kMaxSplits = kAttendFewSplits;

// Four int32 values as balanced base-256 digits: byte d of (x + 0x808080) ^
// 0x808080 is digit d in [-128, 127].  Returns byte `digit` of each, packed;
// `pick` is digit | (4 + digit) << 8.
__device__ __forceinline__ int digits4(int x0, int x1, int x2, int x3, uint32_t pick) {
    constexpr int kBias = 0x00808080;
    const uint32_t w0 = static_cast<uint32_t>((x0 + kBias) ^ kBias), w1 = static_cast<uint32_t>((x1 + kBias) ^ kBias);
    const uint32_t w2 = static_cast<uint32_t>((x2 + kBias) ^ kBias), w3 = static_cast<uint32_t>((x3 + kBias) ^ kBias);
    const uint32_t lo = __builtin_amdgcn_perm(w1, w0, pick), hi = __builtin_amdgcn_perm(w3, w2, pick);
    return static_cast<int>(__builtin_amdgcn_perm(hi, lo, 0x05040100u));
}

// The sum over a quad, the same bits in its four lanes: they hold the digits of
// one weight, and a last place between them would be a carry in one digit and
// not in the next.  So no addition may be fused with the product before it,
// which each lane would round differently.
__device__ __forceinline__ float quad_sum(float v) {
#pragma clang fp contract(off)
    v += dpp<kDppXor1>(v);
    v += dpp<kDppXor2>(v);
    return v;
}

// Element `digit` (the lane's place in its quad) of the quad's sum of v.
__device__ __forceinline__ float quad_sum_pick(f32x4 v, int digit) {
    const bool b0 = digit & 1, b1 = digit & 2;
    float x = b0 ? v[1] : v[0], y = b0 ? v[3] : v[2];
    x += dpp<kDppXor1>(b0 ? v[0] : v[1]);
    y += dpp<kDppXor1>(b0 ? v[2] : v[3]);
    float z = b1 ? y : x;
    z += dpp<kDppXor2>(b1 ? x : y);
    return z;
}

template <int D, int QT>
struct FewState {
    static constexpr int KS = D / 64, DT = D / 16;
    i32x4 q[QT][KS];     // q digits
    float q_scale[QT];   // base-2 score = q_scale * (k scale) * integer product
    int position[QT];    // of the lane's row
    float m[QT], l[QT];  // running maximum; the lane's part of the running sum
    f32x4 o[QT][DT];
    float weight;        // 256^digit
    uint32_t pick;
};

// A block's operands: K and V of a full block, or two planes of the open one.
template <int D>
struct FewTiles {
    i32x4 a[D / 16], b[D / 16];
};
template <int D>
__device__ __forceinline__ void load_tiles(i32x4 (&x)[D / 16], const int8_t *tile) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) x[i] = load16(tile + (i * 64 + (threadIdx.x & 63)) * 16);
}

// Products of K's 16-token tile t with the rows' digits.
template <int D, int QT>
__device__ __forceinline__ i32x4 few_scores(const FewState<D, QT> &st, const i32x4 (&k)[D / 16], int qt, int t) {
    i32x4 c = {0, 0, 0, 0};
#pragma unroll
    for (int x = 0; x < D / 64; ++x)
        c = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[t * (D / 64) + x], st.q[qt][x], c, 0, 0, 0);
    return c;
}

// Bits 4 t + i of the tokens 16 t + i (t, i < 4) that are at most `ahead`.
__device__ __forceinline__ uint32_t first_tokens(int ahead) {
    const int count = ahead < 0 ? 0 : ahead >= 51 ? 16 : ahead / 16 * 4 + min(ahead % 16 + 1, 4);
    return (1u << count) - 1u;
}
// The lane's tokens of the block from `start` on that its row sees: bit 4 t + i
// is token start + 16 t + 4 group + i.
__device__ __forceinline__ uint32_t seen_tokens(int position, int start, uint32_t window) {
    const int ahead = position - start - 4 * ((static_cast<int>(threadIdx.x) & 63) >> 4);
    uint32_t seen = first_tokens(ahead);
    if (window != 0) seen &= ~first_tokens(static_cast<int>(max(static_cast<int64_t>(ahead) - window, static_cast<int64_t>(-1))));
    return seen;
}
// All ones where bit i is set.
__device__ __forceinline__ uint32_t bit_mask(uint32_t bits, int i) {
    return static_cast<uint32_t>(static_cast<int32_t>(bits << (31 - i)) >> 31);
}
// -inf where a bit is clear; bit operations, since compares would each hold a
// pair of scalar registers.
__device__ __forceinline__ void hide(float (&s)[4][4], uint32_t seen) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t m = bit_mask(seen, 4 * t + i);
            s[t][i] = __uint_as_float((__float_as_uint(s[t][i]) & m) | (__float_as_uint(kNegInf) & ~m));
        }
}

// A weight in [0, 1] as 30-bit fixed point.  (A 2^30 inside the exponential
// would cost its argument four bits.)
__device__ __forceinline__ int fixed30(float p) { return static_cast<int>(p * 0x1p30f); }

// The softmax of a block: s holds the lane's base-2 scores (-inf where hidden),
// on return p relative to the block's maximum.  Updates the running maximum and
// sum and rescales o; returns the block's factor relative to the new maximum,
// zero where the row sees nothing of the block.
template <int QT, int DT>
__device__ __forceinline__ float softmax_block(float (&s)[4][4], float &m, float &l, f32x4 (&o)[DT]) {
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[t][i]);
    top = max_xor32(max_xor16(top));
    const float next = fmaxf(m, top);
    const float ref = next == kNegInf ? 0.0f : next;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    const float factor = __builtin_amdgcn_exp2f(top - ref);
    const float shift = top == kNegInf ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[t][i] = __builtin_amdgcn_exp2f(s[t][i] - shift);
            sum += s[t][i];
        }
    l = l * alpha + sum * factor;
    m = next;
    // The maximum seldom moves after the first blocks.  (With two tiles the
    // branch costs more than the products: the accumulators' copies across it
    // would not fit the registers.)
    if (QT > 1 || __builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= alpha;
    }
    return factor;
}

// o += w * (V tile) p
template <int D>
__device__ __forceinline__ void add_values(f32x4 (&o)[D / 16], const i32x4 (&v)[D / 16], i32x4 p, float w) {
    const i32x4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
        const i32x4 c = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[d], p, zero, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][i] = fmaf(static_cast<float>(c[i]), w, o[d][i]);
        if (d % 4 == 3) tile_end();
    }
}

// The open block: codes in two planes, scales per token.  K's token scales
// multiply the scores; V's are folded into the weights, which become fixed point
// relative to the largest product of the two that the row sees.
template <int D, int QT>
__device__ __forceinline__ void few_open_block(FewState<D, QT> &st, const int8_t *planes, const float *scales, int start,
                                               uint32_t window) {
    constexpr size_t kPlane = kKvBlock * D;
    const int group = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        i32x4 high[D / 16], low[D / 16];
        load_tiles<D>(high, planes);
        load_tiles<D>(low, planes + kPlane);
        const uint32_t seen = seen_tokens(st.position[qt], start, window);
        const float unit = st.weight * st.q_scale[qt];
        float s[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const f32x4 ks = *(gptr_f32x4)(uintptr_t)(scales + 16 * t + 4 * group);
            const i32x4 h = few_scores(st, high, qt, t), l = few_scores(st, low, qt, t);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                s[t][i] = quad_sum(fmaf(static_cast<float>(h[i]), 256.0f, static_cast<float>(l[i])) * unit) * ks[i];
        }
        hide(s, seen);
        tile_end();
        load_tiles<D>(high, planes + 2 * kPlane);
        load_tiles<D>(low, planes + 3 * kPlane);
        const float factor = softmax_block<QT>(s, st.m[qt], st.l[qt], st.o[qt]);
        float most = 0.0f, poison = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const f32x4 vs = *(gptr_f32x4)(uintptr_t)(scales + 64 + 16 * t + 4 * group);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float scale = __uint_as_float(__float_as_uint(vs[i]) & bit_mask(seen, 4 * t + i));
                poison += scale - scale;  // NaN where a seen scale is not finite
                s[t][i] *= scale;
                most = fmaxf(most, s[t][i]);
            }
        }
        most = max_xor32(max_xor16(most));
        poison = add_xor32(add_xor16(poison));
        const float inv = most >= 0x1p-126f ? 1.0f / most : 0.0f;  // (32512 of less is under 1e-30, which reads as zero)
        i32x4 p;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            int x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = fixed30(s[t][i] * inv);
            p[t] = digits4(x[0], x[1], x[2], x[3], st.pick);
        }
        const float w = most * factor * (st.weight * 0x1p-30f) + poison;
        add_values<D>(st.o[qt], high, p, 256.0f * w);
        add_values<D>(st.o[qt], low, p, w);
        tile_end();
    }
}

// The rows' q: four rows per tile, column 4 r + digit; a lane has 16 numbers
// of each 64.
template <int D, int QT>
struct FewQuery {
    float x[QT][D / 64][16];
};
template <int D, int QT, typename T>
__device__ __forceinline__ void load_q(FewQuery<D, QT> &q, FewState<D, QT> &st, const AttendArgs &a, const Seq &s, uint32_t head,
                                       int first_row, int rows) {
    const int lane = threadIdx.x & 63, column = lane & 15, group = lane >> 4;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int row = first_row + 4 * qt + (column >> 2);
        const bool live = row < rows;
        const int token = live ? row / static_cast<int>(a.group) : 0;
        const uint32_t h = head * a.group + (live ? row - token * a.group : 0);
        st.position[qt] = s.past + token;
        const T *p = static_cast<const T *>(a.d.q.data) + static_cast<int64_t>(s.first + token) * a.d.q.token_stride +
                     h * a.d.q.head_stride + 16 * group;
#pragma unroll
        for (int k = 0; k < D / 64; ++k) load_floats<T, 16>(p + 64 * k, a.wide != 0, q.x[qt][k]);
    }
}
template <int D, int QT>
__device__ __forceinline__ void digits_of_q(const FewQuery<D, QT> &q, FewState<D, QT> &st, float scale) {
    constexpr int KS = D / 64;
    const int digit = threadIdx.x & 3;
    st.pick = digit | ((4 + digit) << 8);
    st.weight = static_cast<float>(1u << (8 * digit));
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(q.x[qt][k][e]) & 0x7fffffffu);
        top = __float_as_uint(max_xor32(max_xor16(__uint_as_float(min(top, 0x7f800000u)))));  // NaN as infinity
        const bool finite = top < 0x7f800000u;
        // largest = f * 2^e, f in [0.5, 1): q * 2^(30 - e) stays below 2^30.
        const int e2 = __builtin_amdgcn_frexp_expf(__uint_as_float(top));
        const int up = finite && top != 0 ? 30 - e2 : 0;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                int v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = finite ? static_cast<int>(__builtin_amdgcn_ldexpf(q.x[qt][k][4 * w + e], up)) : 0;
                st.q[qt][k][w] = digits4(v[0], v[1], v[2], v[3], st.pick);
            }
        st.q_scale[qt] = finite ? __builtin_amdgcn_ldexpf(scale * kLog2e, -up) : __builtin_nanf("");
    }
    tile_end();
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        st.m[qt] = kNegInf;
        st.l[qt] = 0.0f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) st.o[qt][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
}

// What a workgroup does: one of `splits` parts of a row group's blocks.
struct FewItem {
    int seq;  // -1: nothing
    Seq s;
    uint32_t head, row_group;
    int split, splits;  // `splits` as the sequence's rule gives it
    uint32_t first;     // workgroup of split 0; split i is `step` * i further on
    uint32_t step;
};

// The blocks that rows first_row .. last_row of a sequence see.
struct Span {
    int block0, blocks;
};
__device__ __forceinline__ Span span_of(const AttendArgs &a, int past, int first_row, int last_row) {
    const int group = static_cast<int>(a.group), size = static_cast<int>(kKvBlock);
    const int end = past + last_row / group + 1, position = past + first_row / group;
    const int begin = a.d.window != 0 && static_cast<uint32_t>(position) >= a.d.window
                          ? position - static_cast<int>(a.d.window) + 1 : 0;
    Span s;
    s.block0 = begin / size;
    s.blocks = (end + size - 1) / size - s.block0;
    return s;
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
__device__ __forceinline__ uint64_t wave_total(uint64_t v) {  // v < 2^42
    const uint32_t low = wave_scan(static_cast<uint32_t>(v & 0xffffu)), high = wave_scan(static_cast<uint32_t>(v >> 16));
    return (static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(high, 63))) << 16) +
           static_cast<uint32_t>(__builtin_amdgcn_readlane(low, 63));
}

// What a sequence's workgroups take: every row group of every head is cut into
// parts of about `chunk` blocks (parts_of).
struct SeqWork {
    Seq s;
    uint32_t jobs, blocks;
};
template <int ROWS>
__device__ __forceinline__ SeqWork work_of(const AttendArgs &a, uint32_t i) {
    SeqWork w;
    w.jobs = w.blocks = 0;
    w.s = seq_of(a.batch, a.cache, min(i, a.batch.sequences - 1));
    const uint64_t rows = static_cast<uint64_t>(w.s.count) * a.group;
    if (i >= a.batch.sequences || !w.s.ok || rows == 0 || rows > a.few_rows) return w;
    const uint32_t row_groups = (static_cast<uint32_t>(rows) + ROWS - 1) / ROWS;
    w.jobs = row_groups * a.cache.kv_heads;
    // its longest row group's: the first one with a window, else the last
    w.blocks = max(span_of(a, w.s.past, 0, min(ROWS, static_cast<int>(rows)) - 1).blocks,
                   span_of(a, w.s.past, static_cast<int>(row_groups - 1) * ROWS, static_cast<int>(rows) - 1).blocks);
    return w;
}

// Parts of a row group.  Joining costs 3 us, and 0.1 us more per part; a wave's
// block 2 us, up to where the memory is busy.  So up to kAttendWhole blocks are
// one part, and longer rows have parts of 8, from kAttendLong blocks on of 16
// blocks at least (a token behind, 8 and 16 at least: 1000 tokens 10.5, 9.4 us;
// 4000 11.2, 13.3; 8000 13.1, 13.7; 16000 16.8, 15.5; 32 times 1000 tokens 20.2, 16.9).
__device__ __forceinline__ uint32_t parts_of(uint32_t blocks, uint32_t chunk, uint32_t most) {
    const uint32_t least = blocks <= kAttendWhole || blocks > kAttendLong ? 16 : 8;
    chunk = max(chunk, least);
    return min((blocks + chunk - 1) / chunk, most);
}

// The item of workgroup x.  The device knows the sequences' lengths and the
// host does not, so the deal happens here: all blocks over `target` workgroups,
// and a prefix sum over the sequences, 64 at a time, by every wave for itself.
template <int ROWS>
__device__ __forceinline__ FewItem find_item(const AttendArgs &a, uint32_t x) {
    FewItem it;
    it.seq = -1;
    const int lane = threadIdx.x & 63;
    const uint32_t heads = a.cache.kv_heads;
    if (a.splits == 1) {  // as many workgroups as there may be row groups
        const uint32_t per = a.row_groups * heads;
        it.seq = static_cast<int>(x / per);
        it.s = seq_of(a.batch, a.cache, x / per);
        it.row_group = x % per / heads;
        it.head = x % heads;
        it.split = 0;
        it.splits = 1;
        it.first = x;
        it.step = 1;
        return it;
    }
    SeqWork w;
    uint64_t all = 0;
    for (uint32_t i = 0; i < a.batch.sequences; i += 64) {
        w = work_of<ROWS>(a, i + lane);
        all += wave_total(static_cast<uint64_t>(w.jobs) * w.blocks);
    }
    const uint64_t share = all + a.target - 1;
    uint32_t chunk = share >> 32 == 0 ? static_cast<uint32_t>(share) / a.target : static_cast<uint32_t>(share / a.target);
    // A short last part wastes a workgroup's place: take larger ones until all
    // of them run at once, if they can.
    if (a.batch.sequences <= 64) {
        const uint32_t jobs = __builtin_amdgcn_readlane(wave_scan(w.jobs), 63);
        while (jobs < a.target && static_cast<uint32_t>(__builtin_amdgcn_readlane(
                                      wave_scan(w.jobs * parts_of(w.blocks, chunk, a.splits)), 63)) > a.target)
            chunk += chunk / 8 + 1;
    }
    uint32_t base = 0;
    for (uint32_t i = 0; i < a.batch.sequences; i += 64) {
        if (a.batch.sequences > 64) w = work_of<ROWS>(a, i + lane);
        const uint32_t parts = parts_of(w.blocks, chunk, a.splits), end = base + wave_scan(w.jobs * parts);
        const uint64_t later = __builtin_amdgcn_ballot_w64(end > x);
        if (later != 0) {
            const int owner = __builtin_ctzll(later);
            const uint32_t mine = __builtin_amdgcn_readlane(parts, owner);
            const uint32_t local = x - __builtin_amdgcn_readlane(end - w.jobs * parts, owner);  // (row group, part, head)
            it.seq = static_cast<int>(i) + owner;
            it.s.first = __builtin_amdgcn_readlane(w.s.first, owner);
            it.s.count = __builtin_amdgcn_readlane(w.s.count, owner);
            it.s.past = __builtin_amdgcn_readlane(w.s.past, owner);
            it.s.slot = __builtin_amdgcn_readlane(w.s.slot, owner);
            it.s.length = it.s.past + it.s.count;
            it.s.ok = true;
            it.head = local % heads;
            it.split = static_cast<int>(local / heads % mine);
            it.row_group = local / heads / mine;
            it.splits = static_cast<int>(mine);
            it.step = heads;
            it.first = x - it.split * heads;
            return it;
        }
        base = __builtin_amdgcn_readlane(end, 63);
    }
    return it;
}

template <int D, int QT, int WAVES, typename T>
__global__ __launch_bounds__(64 * WAVES, 2) void attend_few_kernel(const AttendArgs a) {
    constexpr int DT = D / 16, ROWS = 4 * QT, kThreads = 64 * WAVES;
    __shared__ float part[WAVES][ROWS][D];  // the waves' results, then the splits' factors
    static_assert(WAVES * D >= kMaxSplits && kMaxSplits == 64, "they fit; a lane each");
    __shared__ float stat[WAVES][ROWS][2];
    __shared__ uint32_t ticket;

    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const FewItem it = find_item<ROWS>(a, blockIdx.x);
    if (blockIdx.x == 0)  // bad entries, once
        for (uint32_t i = tid; i < a.batch.sequences; i += kThreads)
            if (!seq_of(a.batch, a.cache, i).ok) count_fault(a.cache);
    if (it.seq < 0 || !it.s.ok) return;
    const uint32_t head = it.head;
    const Seq &s = it.s;
    const int rows = s.count * static_cast<int>(a.group);
    const int first_row = it.row_group * ROWS;
    if (first_row >= rows || static_cast<uint32_t>(rows) > a.few_rows) return;
    const int last_row = min(first_row + ROWS, rows) - 1;
    const Span span = span_of(a, s.past, first_row, last_row);
    const int splits = min(it.splits, (span.blocks + WAVES - 1) / WAVES), split = it.split;
    if (split >= splits) return;
    const int from = span.block0 + static_cast<int>(mul_div(split, span.blocks, splits));
    const int to = span.block0 + static_cast<int>(mul_div(split + 1, span.blocks, splits));
    const int open_block = s.length % static_cast<int>(kKvBlock) != 0 ? s.length / static_cast<int>(kKvBlock) : -1;

    // The wave's blocks: from + wave, from + wave + WAVES, ...  Lane x keeps
    // the page of the x-th of the next 64.
    const int32_t *table = a.batch.table + static_cast<size_t>(it.seq) * a.batch.table_width;
    const int mine = to - from > wave ? (to - from - wave + WAVES - 1) / WAVES : 0;
    const bool open_mine = open_block >= from && open_block < to && (open_block - from) % WAVES == wave;
    const int full = mine - (open_mine ? 1 : 0);  // the open block is the sequence's last
    int pages = 0;
    FewTiles<D> tiles;
    f32x2 scale;
    bool bad = false;
    const int8_t *tile = nullptr;
    auto next_tile = [&](int n) {
        if (n % 64 == 0 && n != 0) pages = table[min(from + wave + WAVES * (n + lane), to - 1)];
        int page = __builtin_amdgcn_readlane(pages, n % 64);
        bad = static_cast<uint32_t>(page) >= a.cache.page_count;
        if (bad) {
            if (lane == 0) count_fault(a.cache);
            page = 0;
        }
        tile = a.cache.pages + page_tile(a.cache, page, head);
        scale = *(gptr_f32x2)(uintptr_t)(a.cache.scales + (static_cast<size_t>(page) * a.cache.kv_heads + head) * 2);
    };
    // q's loads go out with the table's and come back before the tiles.
    FewState<D, QT> st;
    FewQuery<D, QT> q;
    if (full > 0) pages = table[min(from + wave + WAVES * lane, to - 1)];
    load_q<D, QT, T>(q, st, a, s, head, first_row, rows);
    tile_end();
    if (full > 0) {
        next_tile(0);
        load_tiles<D>(tiles.a, tile);
        load_tiles<D>(tiles.b, tile + kKvBlock * D);
    }
    tile_end();
    digits_of_q<D, QT>(q, st, a.d.scale);
    const int first_position = s.past + first_row / static_cast<int>(a.group);
    const int last_position = s.past + last_row / static_cast<int>(a.group);
    const int column = lane & 15, group = lane >> 4, digit = column & 3;

    // K's registers take the next block's K as soon as the last scores are out,
    // and V's the next V after the last product: there are always 8 KB in flight.
    for (int n = 0; n < full; ++n) {
        const int start = (from + wave + WAVES * n) * static_cast<int>(kKvBlock);
        const bool masked = start + static_cast<int>(kKvBlock) - 1 > first_position ||
                            (a.d.window != 0 && static_cast<uint32_t>(last_position - start) >= a.d.window);
        const float k_scale = bad ? __builtin_nanf("") : scale[0], v_scale = bad ? __builtin_nanf("") : scale[1];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            float s4[4][4];
            const float w = st.weight * (st.q_scale[qt] * k_scale);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const i32x4 c = few_scores(st, tiles.a, qt, t);
#pragma unroll
                for (int i = 0; i < 4; ++i) s4[t][i] = quad_sum(static_cast<float>(c[i]) * w);
            }
            tile_end();
            if (qt == QT - 1 && n + 1 < full) {
                next_tile(n + 1);
                load_tiles<D>(tiles.a, tile);
            }
            tile_end();
            if (masked) hide(s4, seen_tokens(st.position[qt], start, a.d.window));
            const float factor = softmax_block<QT>(s4, st.m[qt], st.l[qt], st.o[qt]);
            i32x4 p;
#pragma unroll
            for (int t = 0; t < 4; ++t)
                p[t] = digits4(fixed30(s4[t][0]), fixed30(s4[t][1]), fixed30(s4[t][2]), fixed30(s4[t][3]), st.pick);
            // A row that sees nothing of the block takes nothing of it, a NaN scale included.
            const float wv = masked && factor == 0.0f ? 0.0f : v_scale * factor * (st.weight * 0x1p-30f);
            tile_end();
            add_values<D>(st.o[qt], tiles.b, p, wv);
        }
        if (n + 1 < full) load_tiles<D>(tiles.b, tile + kKvBlock * D);
        tile_end();
    }
    if (open_mine)
        few_open_block<D, QT>(st, a.cache.open + open_tile(a.cache, s.slot, open_block, head),
                              a.cache.open_scales + open_scale_row(a.cache, s.slot, open_block, head),
                              open_block * static_cast<int>(kKvBlock), a.d.window);

    // Join the digits and the lanes' sums, then the waves.
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int r = 4 * qt + (column >> 2);
        const float l = add_xor32(add_xor16(st.l[qt]));
        if (group == 0 && digit == 0) {
            stat[wave][r][0] = st.m[qt];
            stat[wave][r][1] = l;
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) part[wave][r][16 * d + 4 * group + digit] = quad_sum_pick(st.o[qt][d], digit);
    }
    __syncthreads();

    const int live_rows = min(ROWS, rows - first_row);
    const auto finish = [&](int r, int d, float m, float l, float o) {
        const int row = first_row + r, token = row / static_cast<int>(a.group);
        const uint32_t h = head * a.group + (row - token * a.group);
        static_cast<T *>(a.d.out.data)[static_cast<int64_t>(s.first + token) * a.d.out.token_stride +
                                       h * a.d.out.head_stride + d] = static_cast<T>(l == 0.0f ? 0.0f : o / l);
        if (d == 0 && a.d.lse != nullptr)
            a.d.lse[static_cast<size_t>(s.first + token) * a.d.q_heads + h] = (m + log2f(l)) * (1.0f / kLog2e);
    };
    float *stats = a.partials + static_cast<size_t>(gridDim.x) * ROWS * D;
    const size_t slot = static_cast<size_t>(blockIdx.x) * ROWS;
    for (int x = tid; x < live_rows * D; x += kThreads) {
        const int r = x / D, d = x % D;
        float m = kNegInf;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) m = fmaxf(m, stat[w][r][0]);
        const float ref = m == kNegInf ? 0.0f : m;
        float l = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f(stat[w][r][0] - ref);
            l += stat[w][r][1] * f;
            o += part[w][r][d] * f;
        }
        if (splits > 1) {
            store_agent(a.partials + (slot + r) * D + d, o);
            if (d == 0) {
                store_agent(stats + (slot + r) * 2, m);
                store_agent(stats + (slot + r) * 2 + 1, l);
            }
        } else {
            finish(r, d, m, l, o);
        }
    }
    if (splits == 1) return;

    // The last workgroup of the row group joins the splits.
    wait_stores();
    __syncthreads();
    uint32_t *arrived = a.arrived + (static_cast<size_t>(it.seq) * a.row_groups + it.row_group) * a.cache.kv_heads + head;
    if (tid == 0) ticket = add_agent(arrived, 1u);
    __syncthreads();
    if (ticket != static_cast<uint32_t>(splits - 1)) return;
    if (tid == 0) store_agent(arrived, 0u);
    // The partial results go out first, all at once: one trip to the memory
    // behind the L2s.  Meanwhile each wave turns its rows' statistics, a split
    // per lane, into the splits' factors.
    constexpr int kPairs = ROWS * D / 2, kRounds = kPairs > kThreads ? kPairs / kThreads : 1;
    const size_t first_slot = it.first;
    float(*factor)[kMaxSplits] = reinterpret_cast<float(*)[kMaxSplits]>(&part[0][0][0]);
#pragma unroll
    for (int round = 0; round < kRounds; ++round) {
        const int x = tid + kThreads * round, r = x / (D / 2), d = x % (D / 2) * 2;
        const bool live = x < live_rows * (D / 2);
        f32x2 v[kMaxSplits];
        if (live) {
#pragma unroll
            for (int i0 = 0; i0 < kMaxSplits; i0 += 8)
                if (i0 < splits) {
#pragma unroll
                    for (int i = i0; i < i0 + 8; ++i)
                        v[i] = load_agent2(a.partials + ((first_slot + min(i, splits - 1) * it.step) * ROWS + r) * D + d);
                }
        }
        if (round == 0) {
            for (int y = wave; y < ROWS; y += WAVES) {
                f32x2 ml = {kNegInf, 0.0f};
                if (lane < splits) ml = load_agent2(stats + ((first_slot + lane * it.step) * ROWS + y) * 2);
                float m = ml[0];
                m = fmaxf(m, dpp<kDppXor1>(m));
                m = fmaxf(m, dpp<kDppXor2>(m));
                m = fmaxf(m, dpp<kDppMirror8>(m));
                m = fmaxf(m, dpp<kDppMirror16>(m));
                m = max_xor32(max_xor16(m));
                const float f = __builtin_amdgcn_exp2f(ml[0] - (m == kNegInf ? 0.0f : m));
                const float l = add_xor32(add_xor16(lanes_sum<16>(ml[1] * f)));
                factor[y][lane] = f;
                if (lane == 0) {
                    stat[0][y][0] = m;
                    stat[0][y][1] = l;
                }
            }
            __syncthreads();
        }
        if (live) {
            float o0 = 0.0f, o1 = 0.0f;
#pragma unroll
            for (int i0 = 0; i0 < kMaxSplits; i0 += 8)
                if (i0 < splits) {
#pragma unroll
                    for (int i = i0; i < i0 + 8; ++i)
                        if (i < splits) {
                            o0 += v[i][0] * factor[r][i];
                            o1 += v[i][1] * factor[r][i];
                        }
                }
            finish(r, d, stat[0][r][0], stat[0][r][1], o0);
            finish(r, d + 1, stat[0][r][0], stat[0][r][1], o1);
        }
    }
}

template <int WAVES, typename T>
void launch_few(const AttendArgs &a, uint32_t rows, hipStream_t stream) {
    auto go = [&](auto kernel) { kernel<<<a.workgroups, 64 * WAVES, 0, stream>>>(a); };
    if (a.cache.head_dim == 64)
        rows == 4 ? go(attend_few_kernel<64, 1, WAVES, T>) : go(attend_few_kernel<64, 2, WAVES, T>);
    else
        rows == 4 ? go(attend_few_kernel<128, 1, WAVES, T>) : go(attend_few_kernel<128, 2, WAVES, T>);
}
template <typename T>
void launch_few(const AttendArgs &a, uint32_t rows, uint32_t waves, hipStream_t stream) {
    waves == 4 ? launch_few<4, T>(a, rows, stream) : launch_few<8, T>(a, rows, stream);
}

}  // namespace

uint32_t attend_few_rows(uint32_t rows) { return rows <= 4 ? 4 : 8; }

hipError_t launch_attend_few(const AttendArgs &a, uint32_t rows, uint32_t waves, hipStream_t stream) {
    if (a.d.dtype == Q4RDNA_F32) launch_few<float>(a, rows, waves, stream);
    else if (a.d.dtype == Q4RDNA_F16) launch_few<_Float16>(a, rows, waves, stream);
    else launch_few<__bf16>(a, rows, waves, stream);
    return hipGetLastError();
}

}  // namespace q4rdna
